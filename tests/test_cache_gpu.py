"""The paged 8-bit cache on the GPU against the 64-bit oracle (oracle/cache.py).

``cache_append`` is compared for equality: stored bytes, scales and the rotated q are roundings of
exact values.  ``cache_attention`` is compared within the room that the oracle derives from the
kernels' roundings, plus half a step of the output's type.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

import fused_attn
from oracle import cache as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _available():
    if not fused_attn.is_available() or not fused_attn.impl_supports(5, torch.float16, 128):
        pytest.skip("kernels not available")
    fused_attn.last_device_error()
    yield


class Setup:
    """A cache with a batch over it: `lens` keys held after the step, `new` tokens each."""

    def __init__(self, lens, new, H=4, Hkv=2, D=128, page=16, dtype=torch.bfloat16, seed=0, rot=None,
                 token_major=False, tail=0, spare=3, uniform=False, strided=False):
        g = torch.Generator().manual_seed(seed)
        self.g, self.H, self.Hkv, self.D, self.page, self.dtype = g, H, Hkv, D, page, dtype
        self.lens, self.new = list(lens), list(new)
        S, counts = len(self.lens), [-(-max(n, 0) // page) for n in lens]
        P = sum(counts) + spare
        order = torch.randperm(P, generator=g)
        width = max([1, *counts])
        table = torch.full((S, width), -7, dtype=torch.int32)  # entries that are not to be read
        at = 0
        for s, n in enumerate(counts):
            table[s, :n] = order[at:at + n]
            at += n
        self.table, self.P = table, P
        shape = (P, page, Hkv, D) if token_major else (P, Hkv, page, D)

        def pool(spread):
            x = torch.randn(shape, generator=g) * 3
            scale = torch.exp2(torch.randint(-spread, spread + 1, (P, Hkv), generator=g).float())
            c = x.to(E4M3).cuda()
            return (c.transpose(1, 2) if token_major else c), scale.cuda()

        self.k_cache, self.k_scale = pool(2)
        self.v_cache, self.v_scale = pool(4)
        T = sum(self.new) + tail
        rows = torch.randn(T, H + 2 * Hkv, D, generator=g)
        rows = rows.to(dtype).cuda()
        if strided:
            self.q, self.k, self.v = rows.split([H, Hkv, Hkv], 1)
        else:
            self.q, self.k, self.v = (x.contiguous() for x in rows.split([H, Hkv, Hkv], 1))
        self.table_d = table.cuda()
        self.lens_d = torch.tensor(self.lens, dtype=torch.int32).cuda()
        cu = [0]
        for n in self.new:
            cu.append(cu[-1] + n)
        self.cu = None if uniform else cu
        self.cu_d = None if uniform else torch.tensor(cu, dtype=torch.int32).cuda()
        self.cos = self.sin = None
        if rot:
            pos = torch.arange(max([1, *self.lens]), dtype=torch.float64)
            angle = pos[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
            self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()

    def pages(self):
        return ref.pages_of(self.k_cache, self.v_cache, self.k_scale, self.v_scale)

    def append(self, with_q=True, interleaved=False):
        return fused_attn.cache_append(
            self.k, self.v, self.k_cache, self.v_cache, self.k_scale, self.v_scale, self.table_d,
            self.lens_d, cu_seqlens=self.cu_d, q=self.q if with_q and self.cos is not None else None,
            cos=self.cos, sin=self.sin, interleaved=interleaved)

    def attend(self, causal=True, scale=None, q=None):
        return fused_attn.cache_attention(
            self.q if q is None else q, self.k_cache, self.v_cache, self.k_scale, self.v_scale,
            self.table_d, self.lens_d, cu_seqlens=self.cu_d, is_causal=causal, scale=scale,
            return_lse=True)


def same_pages(got: ref.Pages, want: ref.Pages):
    for name, a, b in zip(got._fields, got, want):
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        assert torch.equal(a.nan_to_num(), b.nan_to_num()), name


def check_append(s: Setup, interleaved=False, with_q=True, errors=(0, 0)):
    want = s.pages()
    q_want = ref.append(want, s.k, s.v, s.table.tolist(), s.lens, s.cu, q=s.q if s.cos is not None and with_q else None,
                        cos=s.cos, sin=s.sin, interleaved=interleaved)
    q = s.append(interleaved=interleaved, with_q=with_q)
    torch.cuda.synchronize()
    same_pages(s.pages(), want)
    if q_want is None:
        assert q is None
    else:
        # fp32 holds the rounding to odd, so the rounding to 16 bits is the exact value's
        assert torch.equal(q.cpu(), narrow(q_want, s.dtype))
    assert fused_attn.last_device_error() == errors


def narrow(x: torch.Tensor, dtype) -> torch.Tensor:
    """float64 to fp16 / bf16 with one rounding."""
    m, e = torch.frexp(x)
    bits, low = (11, -14) if dtype == torch.float16 else (8, -126)
    step = torch.exp2((torch.clamp(e - 1, min=low) - (bits - 1)).double())
    return (torch.round(x / step) * step).to(dtype)


def check_attention(s: Setup, causal=True, scale=None, o=None, lse=None):
    if o is None:
        o, lse = s.attend(causal, scale)
    want = ref.attention(s.pages(), s.q, s.table.tolist(), s.lens, s.cu, causal, scale)
    o, lse = o.cpu().double(), lse.cpu().double()
    fin = torch.isfinite(want.lse)
    assert torch.equal(torch.isfinite(lse), fin) and bool((lse[~fin] == math.inf).all())
    assert bool(((lse - want.lse)[fin].abs() <= want.lse_room[fin]).all()), \
        float(((lse - want.lse)[fin].abs() / want.lse_room[fin].clamp(min=1e-12)).max())
    half = torch.finfo(s.dtype).eps / 2
    tiny = torch.finfo(s.dtype).smallest_normal * half
    room = want.o_room * (1 + half) + want.o.abs() * half + tiny
    assert bool(((o - want.o).abs() <= room).all()), float(((o - want.o).abs() / room).max())
    assert fused_attn.last_device_error() == (0, 0)


# ---- append ----


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("rot,interleaved", [(None, False), (128, False), (128, True), (32, False), (48, True),
                                             (16, False)])
@pytest.mark.parametrize("D", [64, 128])
def test_append_rotations(D, rot, interleaved, dtype):
    if rot and rot > D:
        rot = D
    s = Setup([5, 40, 17, 64], [5, 3, 17, 40], D=D, dtype=dtype, rot=rot, seed=1, strided=True)
    check_append(s, interleaved)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([130], [130]), ([129, 1, 300], [1, 1, 1]),
                                      ([200, 7, 33, 64], [8, 0, 20, 64]), ([257], [256]), ([0, 16, 0], [0, 16, 0])],
                         ids=str)
@pytest.mark.parametrize("token_major", [False, True], ids=["heads", "tokens"])
def test_append_lengths_and_pages(lens, new, page, token_major):
    check_append(Setup(lens, new, page=page, rot=64, D=64, H=3, Hkv=1, seed=2, token_major=token_major, tail=2))


@pytest.mark.parametrize("Hkv,H", [(1, 1), (12, 12), (3, 21), (8, 64)])
@pytest.mark.parametrize("n", [1, 9], ids=["token", "rows"])
def test_append_heads_and_uniform_batches(Hkv, H, n):
    check_append(Setup([n + 3 * i for i in range(7)], [n] * 7, H=H, Hkv=Hkv, rot=128, uniform=True, seed=3))


def test_append_in_steps_grows_the_scale():
    """Rows that get larger: at most steps the page's earlier rows move to a larger step."""
    s = Setup([40], [40], rot=128, seed=4, page=32)
    k, v, q = s.k, s.v, s.q
    want, grown = s.pages(), 0
    at = 0
    for n in (1, 1, 2, 5, 1, 9, 12, 1, 8):
        f = 2.0 ** (at / 2 - 6)
        s.k, s.v, s.q = k[at:at + n] * f, v[at:at + n] * f, q[at:at + n]
        s.lens_d.fill_(at + n)
        before = s.k_scale.clone()
        ref.append(want, s.k, s.v, s.table.tolist(), [at + n], [0, n], cos=s.cos, sin=s.sin)
        s.cu_d.copy_(torch.tensor([0, n]))
        s.append()
        torch.cuda.synchronize()
        same_pages(s.pages(), want)
        grown += int((s.k_scale > before).any())
        at += n
    assert grown >= 4 and fused_attn.last_device_error() == (0, 0)


@pytest.mark.parametrize("n", [1, 30], ids=["token", "rows"])
def test_append_extreme_values(n):
    """The type's largest and smallest values, zero rows, infinities and NaN."""
    for dtype in (torch.float16, torch.bfloat16):
        s = Setup([n, n + 5, n, n], [n] * 4, rot=128, seed=5, dtype=dtype)
        fi = torch.finfo(dtype)
        s.k[0:n] = fi.max
        s.v[0:n] = fi.smallest_normal
        s.k[n:2 * n] = 0
        s.v[n:2 * n] = 0
        s.k[2 * n, 0, 3] = math.inf
        s.v[2 * n, 1, 5] = -math.inf
        s.v[2 * n, 0, 0] = math.nan
        s.k[3 * n:] *= 1e-4
        s.q[0:n] = 0
        want = s.pages()
        ref.append(want, s.k, s.v, s.table.tolist(), s.lens, s.cu, cos=s.cos, sin=s.sin)
        s.append(with_q=False)
        torch.cuda.synchronize()
        got = s.pages()
        same_pages(got, want)
        assert bool(torch.isnan(got.k).any()) and bool(torch.isnan(got.v).any())


def test_append_takes_a_scale_that_is_no_power_of_two_up_to_the_next():
    s = Setup([8], [2], seed=6, page=16)
    s.k_scale.fill_(0.75)
    s.v_scale.fill_(3.0)
    want = s.pages()
    ref.append(want, s.k, s.v, s.table.tolist(), s.lens, s.cu)
    s.append()
    torch.cuda.synchronize()
    same_pages(s.pages(), want)
    assert bool((s.k_scale[s.table[0, 0]] == 1.0).all()) and bool((s.v_scale[s.table[0, 0]] == 4.0).all())


def test_append_leaves_other_pages_and_rows_alone():
    s = Setup([37, 20], [5, 4], rot=64, seed=7, spare=9, tail=6)
    k0, v0 = s.k_cache.view(torch.uint8).clone(), s.v_cache.view(torch.uint8).clone()
    ks0, vs0 = s.k_scale.clone(), s.v_scale.clone()
    q = s.append()
    touched = torch.zeros(s.P, s.page, dtype=torch.bool)
    for seq, (n, m) in enumerate(zip(s.lens, s.new)):
        for pos in range(n):
            if pos // s.page >= (n - m) // s.page:
                touched[s.table[seq, pos // s.page], pos % s.page] = True
    same = ~touched[:, None, :, None].cuda()
    for now, was in ((s.k_cache, k0), (s.v_cache, v0)):
        assert bool(((now.view(torch.uint8) == was) | ~same).all())
    pages = ~touched.any(1).cuda()
    assert torch.equal(s.k_scale[pages], ks0[pages]) and torch.equal(s.v_scale[pages], vs0[pages])
    assert not bool(q[9:].any())


# ---- attention ----


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([15, 16, 17, 63, 64, 65, 129], [1] * 7), ([700, 3], [1, 1]),
                                      ([40, 0, 90, 5], [4, 0, 9, 5]), ([200], [33])], ids=str)
def test_attention_lengths_and_pages(lens, new, page, D, dtype):
    check_attention(Setup(lens, new, page=page, D=D, dtype=dtype, seed=11, tail=1))


@pytest.mark.parametrize("H,Hkv", [(1, 1), (12, 12), (7, 1), (24, 8), (16, 1), (32, 1), (40, 2)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("new", [1, 2, 6, 17])
def test_attention_heads(H, Hkv, new, causal):
    check_attention(Setup([new, 30 + new, 150], [new] * 3, H=H, Hkv=Hkv, D=64, seed=12, uniform=True), causal)


def test_attention_rows_without_keys():
    """More queries than keys (the leading ones see none), and a sequence without keys."""
    s = Setup([2, 0, 5], [6, 3, 5], seed=13)
    o, lse = s.attend()
    check_attention(s, o=o, lse=lse)
    assert bool((lse[:4] == math.inf).all()) and bool((lse[6:9] == math.inf).all()) and not bool(o[:4].any())
    s = Setup([2, 0], [4, 2], seed=13)
    check_attention(s, causal=False)


def test_attention_ignores_what_lies_behind_a_sequence():
    """NaN in every slot behind the last key, in every unused page, and their scales."""
    s = Setup([5, 30, 64, 100], [1, 2, 1, 3], seed=14, page=32)
    o0, lse0 = s.attend()
    used = torch.zeros(s.P, s.page, dtype=torch.bool)
    for seq, n in enumerate(s.lens):
        for pos in range(n):
            used[s.table[seq, pos // s.page], pos % s.page] = True
    dead = ~used[:, None, :, None].expand(s.P, s.Hkv, s.page, s.D).cuda()
    for c, sc in ((s.k_cache, s.k_scale), (s.v_cache, s.v_scale)):
        c.view(torch.uint8).masked_fill_(dead, 0x7F)
        sc[~used.any(1).cuda()] = math.nan
    o, lse = s.attend()
    assert torch.equal(o, o0) and torch.equal(lse, lse0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_attention_scales(dtype):
    """Scales over forty binades, some no powers of two, a page of zeros; large and small queries."""
    s = Setup([333, 64, 90], [3, 1, 2], seed=15, dtype=dtype)
    g = s.g
    s.k_scale.copy_(torch.exp2(4 * torch.randn(s.P, s.Hkv, generator=g) - 8))
    s.v_scale.copy_(torch.exp2(10 * torch.randn(s.P, s.Hkv, generator=g)).clamp(2**-20, 2**20))
    s.v_cache.view(torch.uint8)[s.table[0, 3].item()] = 0
    s.q *= torch.exp2(torch.randint(-12, 3, (s.q.shape[0], s.H, 1), generator=g).float()).cuda().to(dtype)
    # the output must stay in fp16's range for the comparison to mean something
    if dtype == torch.float16:
        s.v_scale.clamp_(max=16.0)
    check_attention(s)


def test_attention_one_large_score():
    """Scores far apart: the running maximum jumps, late and early."""
    for at in (0, 17, 95, 199):
        s = Setup([200], [1], seed=16, D=64)
        page, slot = s.table[0, at // 16].item(), at % 16
        s.k_cache[page, :, slot] = (s.q[0].view(s.Hkv, 2, 64).sum(1).float() * 20).clamp(-448, 448).to(E4M3)
        check_attention(s)


def test_attention_nan_in_a_visible_key_reaches_its_rows_only():
    s = Setup([50, 40], [1, 1], seed=17)
    s.k_cache.view(torch.uint8)[s.table[0, 1].item(), 0, 4] = 0x7F
    o, lse = s.attend()
    assert bool(torch.isnan(o[0, :2]).all()) and bool(torch.isnan(lse[0, :2]).all())
    assert bool(torch.isfinite(o[0, 2:]).all()) and bool(torch.isfinite(o[1]).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,new", [([50, 40], [8, 3]), ([700, 300], [5, 7]), ([300, 180], [200, 60]),
                                      ([2600, 40], [300, 40])])
def test_attention_nan_in_a_value_stays_with_the_rows_that_see_it(lens, new, D):
    """A value that is NaN behind a causal row's own position does not reach it: 0 weights and NaN."""
    s = Setup(lens, new, D=D, seed=27)
    clean_o, clean_lse = s.attend()
    first = 0
    want = torch.zeros(sum(new), s.H, D, dtype=torch.bool)
    group = s.H // s.Hkv
    for i, (length, n) in enumerate(zip(lens, new)):
        for back, head, col in ((n // 2, 0, 5), (1, 1, D - 1), (n - 1, 1, 33)):
            key = length - back  # new token n - back
            s.v_cache.view(torch.uint8)[s.table[i, key // s.page].item(), head, key % s.page, col] = 0xFF
            want[first + n - back:first + n, head * group:(head + 1) * group, col] = True
        first += n
    o, lse = s.attend()
    torch.cuda.synchronize()
    assert torch.equal(torch.isnan(o).cpu(), want)
    assert torch.equal(lse, clean_lse)
    keep = ~want.cuda()
    assert torch.equal(o[keep], clean_o[keep])
    assert fused_attn.last_device_error() == (0, 0)


def test_attention_layouts_agree():
    """Token-major pools, strided q, wider tables: the same numbers, the same bits."""
    a = Setup([100, 37, 260], [2, 1, 5], seed=18)
    o, lse = a.attend()
    wide = torch.empty(a.q.shape[0], 3 * a.H, a.D, dtype=a.dtype, device="cuda")
    view = wide[:, a.H:2 * a.H]
    view.copy_(a.q)
    tm = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (a.k_cache.view(torch.uint8),
                                                                    a.v_cache.view(torch.uint8))]
    table = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    table[:, :a.table.shape[1]] = a.table_d
    o2, lse2 = fused_attn.cache_attention(view, tm[0].view(E4M3), tm[1].view(E4M3), a.k_scale, a.v_scale,
                                          table, a.lens_d, cu_seqlens=a.cu_d, return_lse=True)
    # a wider table may change the number of CTAs and so the order of sums
    ref_ = ref.attention(a.pages(), a.q, a.table.tolist(), a.lens, a.cu)
    half = torch.finfo(a.dtype).eps / 2
    assert bool(((o2.cpu().double() - ref_.o).abs() <= ref_.o_room * 1.01 + ref_.o.abs() * half).all())
    assert bool(((lse2 - lse).abs() <= 1e-4).all())
    o3, lse3 = fused_attn.cache_attention(view, tm[0].view(E4M3), tm[1].view(E4M3), a.k_scale, a.v_scale,
                                          a.table_d, a.lens_d, cu_seqlens=a.cu_d, return_lse=True)
    assert torch.equal(o3, o) and torch.equal(lse3, lse)


@pytest.mark.parametrize("new,H", [(1, 2), (1, 12), (9, 4)])
def test_attention_long_sequences(new, H):
    """Enough keys that each CTA walks many pages of one sequence, against fp64 on the GPU."""
    Hkv, D, page, lens = 1, 64, 16, [1300000, 1234, 5, 600001]
    counts = [-(-n // page) for n in lens]
    P = sum(counts)
    g = torch.Generator(device="cuda").manual_seed(31)
    pools = [torch.randn(P, Hkv, page, D, generator=g, device="cuda").to(E4M3) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-2, 3, (P, Hkv), generator=g, device="cuda").float()) for _ in range(2)]
    order = torch.randperm(P, generator=g, device="cuda").int()
    table = torch.full((4, max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    q = torch.randn(4 * new, H, D, generator=g, device="cuda").half()
    o, lse = fused_attn.cache_attention(q, *pools, *scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                        return_lse=True)
    for s, n in enumerate(lens):
        ids = table[s, :counts[s]].long()
        k, v = (x.view(torch.uint8)[ids].view(E4M3).double() * sc[ids].double()[..., None, None]
                for x, sc in zip(pools, scales))
        k, v = k.reshape(-1, D)[:n], v.reshape(-1, D)[:n]
        for i in range(new):
            seen = max(0, n - new + i + 1)
            a = q[s * new + i].double() @ k[:seen].T / 8
            if seen == 0:
                assert bool((lse[s * new + i] == math.inf).all())
                continue
            want = torch.softmax(a, -1)
            room = want @ v[:seen].abs() * 2.0**-10 + 1e-6
            want_o = want @ v[:seen]
            assert bool(((o[s * new + i].double() - want_o).abs() <= room + want_o.abs() * 2.0**-11).all())
            assert bool(((lse[s * new + i].double() - torch.logsumexp(a, -1)).abs() < 1e-4).all())
    assert fused_attn.last_device_error() == (0, 0)


def test_attention_repeats_bit_for_bit():
    s = Setup([3000, 1, 700, 2500], [1, 1, 3, 40], seed=19, page=64)
    o, lse = s.attend()
    for _ in range(10):
        o2, lse2 = s.attend()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("seed", range(24))
def test_attention_random_batches(seed):
    r = random.Random(seed)
    Hkv = r.choice([1, 2, 4])
    S = r.randint(1, 5)
    new = [r.choice([0, 1, 1, 1, 2, 5, 30]) for _ in range(S)]
    lens = [max(0, n + r.choice([-1, 0, 1, 13, 100, 333])) for n in new]
    s = Setup(lens, new, H=Hkv * r.choice([1, 2, 3, 8]), Hkv=Hkv, D=r.choice([64, 128]),
              page=r.choice([16, 32, 64, 128]), dtype=r.choice([torch.float16, torch.bfloat16]), seed=100 + seed,
              tail=r.choice([0, 2]), token_major=r.random() < 0.3, strided=r.random() < 0.5)
    check_attention(s, causal=r.random() < 0.7, scale=r.choice([None, 0.02, 0.5]))


# ---- the same with many rows a sequence, which another kernel serves ----


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("lens,new", [([300], [300]), ([129, 128, 127], [60, 128, 127]), ([700, 40], [90, 33]),
                                      ([64, 500, 1], [64, 1, 1])], ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_many_rows(lens, new, causal, dtype, D):
    check_attention(Setup(lens, new, H=8, Hkv=2, D=D, dtype=dtype, page=32, seed=41, tail=2), causal)


@pytest.mark.parametrize("H,Hkv", [(3, 3), (7, 1), (130, 1), (300, 1)])
def test_many_rows_groups(H, Hkv):
    """Groups that do not divide a tile, up to more heads than a tile has rows."""
    check_attention(Setup([90, 200], [40, 3], H=H, Hkv=Hkv, D=64, page=64, seed=42, dtype=torch.float16))


def test_many_rows_without_keys():
    s = Setup([20, 0, 50], [60, 40, 50], H=8, Hkv=1, seed=43)
    o, lse = s.attend()
    check_attention(s, o=o, lse=lse)
    assert bool((lse[:40] == math.inf).all()) and bool((lse[60:100] == math.inf).all()) and not bool(o[:40].any())


def test_many_rows_scales_and_garbage():
    """Scales over twenty binades, NaN behind every sequence and in unused pages."""
    s = Setup([333, 64, 200], [30, 64, 41], H=8, Hkv=2, seed=44, page=32, dtype=torch.bfloat16)
    s.k_scale.copy_(torch.exp2(3 * torch.randn(s.P, s.Hkv, generator=s.g) - 8))
    s.v_scale.copy_(torch.exp2(5 * torch.randn(s.P, s.Hkv, generator=s.g)).clamp(2**-10, 2**10))
    used = torch.zeros(s.P, s.page, dtype=torch.bool)
    for seq, n in enumerate(s.lens):
        for pos in range(n):
            used[s.table[seq, pos // s.page], pos % s.page] = True
    dead = ~used[:, None, :, None].expand(s.P, s.Hkv, s.page, s.D).cuda()
    for c, sc in ((s.k_cache, s.k_scale), (s.v_cache, s.v_scale)):
        c.view(torch.uint8).masked_fill_(dead, 0x7F)
        sc[~used.any(1).cuda()] = math.nan
    clean = s.pages()
    for x in clean[:2]:
        x.nan_to_num_()
    for x in clean[2:]:
        x.nan_to_num_(1.0)
    s.pages = lambda: clean
    check_attention(s)


def test_many_rows_long_chunk_against_64_bits():
    """Tiles that several CTAs share, over many key tiles, against fp64 on the GPU."""
    for D, H, Hkv, n, L in ((128, 8, 2, 300, 20000), (64, 4, 1, 77, 90001), (128, 16, 1, 5, 70000)):
        page = 64
        counts = -(-L // page)
        g = torch.Generator(device="cuda").manual_seed(45)
        pools = [torch.randn(counts, Hkv, page, D, generator=g, device="cuda").to(E4M3) for _ in range(2)]
        scales = [torch.exp2(torch.randint(-2, 3, (counts, Hkv), generator=g, device="cuda").float()) for _ in "kv"]
        table = torch.randperm(counts, generator=g, device="cuda").int()[None]
        q = torch.randn(n, H, D, generator=g, device="cuda").bfloat16()
        lens = torch.tensor([L], dtype=torch.int32, device="cuda")
        o, lse = fused_attn.cache_attention(q, *pools, *scales, table, lens, return_lse=True)
        assert fused_attn.last_device_error() == (0, 0)
        ids = table[0].long()
        k, v = ((x.view(torch.uint8)[ids].view(E4M3).double() * sc[ids].double()[..., None, None]).transpose(0, 1)
                .reshape(Hkv, -1, D)[:, :L] for x, sc in zip(pools, scales))
        hidden = torch.arange(L, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + (L - n)
        for h in range(H):
            a = (q[:, h].double() @ k[h * Hkv // H].T / D**0.5).masked_fill_(hidden, -math.inf)
            p = torch.softmax(a, -1)
            want = p @ v[h * Hkv // H]
            room = p @ v[h * Hkv // H].abs() * 2.0**-10 + want.abs() * 2.0**-8 + 1e-6
            assert bool(((o[:, h].double() - want).abs() <= room).all())
            assert bool(((lse[:, h].double() - torch.logsumexp(a, -1)).abs() < 1e-4).all())


def test_many_rows_repeat_bit_for_bit():
    s = Setup([1500, 40, 700], [200, 40, 333], H=8, Hkv=2, seed=46, page=64)
    o, lse = s.attend()
    for _ in range(10):
        o2, lse2 = s.attend()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("new", [1, 40], ids=["tokens", "rows"])
def test_many_sequences(new):
    """More sequences than a block has threads, some without new tokens, some without keys."""
    r = random.Random(7)
    S = 1400
    n = [0 if i % 97 == 5 else r.choice([1, new]) if new > 1 else 1 for i in range(S)]
    lens = [0 if i % 131 == 7 else m + r.choice([0, 3, 150]) for i, m in enumerate(n)]
    s = Setup(lens, n, H=4, Hkv=1, D=64, page=32, rot=64, seed=47, dtype=torch.float16)
    before = s.pages()
    q = s.append()
    s.q = q
    o, lse = s.attend()
    # tokens in front of the cache (sequences that hold nothing) are reported, the others stored
    assert fused_attn.last_device_error()[0] in (0, 1)
    picks = sorted({0, 5, 7, 8, 700, 701, S - 1, *(r.randrange(S) for _ in range(20))})
    after = s.pages()
    for i in picks:
        rows = slice(s.cu[i], s.cu[i + 1])
        sub = [0, s.cu[i + 1] - s.cu[i]]
        table = [s.table[i].tolist()]
        page_ids = [p for p in table[0] if p >= 0]
        want = ref.Pages(*(x.clone() for x in before))
        ref.append(want, s.k[rows], s.v[rows], table, [lens[i]], sub, cos=s.cos, sin=s.sin)
        for a, b in zip(after, want):
            assert torch.equal(a[page_ids], b[page_ids])
        got = ref.attention(after, q[rows], table, [lens[i]], sub)
        half = torch.finfo(torch.float16).eps / 2
        assert bool(((o[rows].cpu().double() - got.o).abs() <= got.o_room * 1.01 + got.o.abs() * half + 1e-7).all())
        fin = torch.isfinite(got.lse)
        assert bool(((lse[rows].cpu().double() - got.lse)[fin].abs() <= got.lse_room[fin]).all())
        assert bool((lse[rows].cpu()[~fin] == math.inf).all())


def test_bad_device_values_with_many_rows():
    def fresh():
        return Setup([120, 233], [64, 50], H=4, Hkv=2, seed=48, page=32)

    for what in ("page", "length", "negative length", "offsets", "offset order"):
        s, good = fresh(), fresh()
        if what == "page":
            s.table_d[0, 1] = s.P
        elif what == "length":
            s.lens_d[0] = 10**6
        elif what == "negative length":
            s.lens_d[0] = -5
        elif what == "offsets":
            s.cu_d[2] = 1000
        elif what == "offset order":
            s.cu_d[0] = 70
        o, _ = s.attend()
        torch.cuda.synchronize()
        assert fused_attn.last_device_error() == (1, 1 << 11), what
        o_good, _ = good.attend()
        if what in ("page", "length", "negative length"):  # the second sequence is as it should be
            assert bool(((o[64:] - o_good[64:]).abs().float() <= 0.02 * o_good[64:].abs().float() + 0.02).all())
        assert fused_attn.last_device_error() == (0, 0)


def test_many_rows_in_a_graph_on_another_stream():
    s = Setup([150, 300], [100, 60], H=8, Hkv=2, rot=128, seed=49, page=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        q = s.append()
        s.attend(q=q)
        with torch.cuda.graph(g, stream=side):
            q = s.append()
            o, lse = s.attend(q=q)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        kept, s.q = s.q, q
        check_attention(s, o=o, lse=lse)
        s.q = kept
    del g


# ---- together, and how they are called ----


def test_prompt_then_tokens_then_a_merge_with_another_part():
    """Prompts appended and attended to, then single tokens; at the end the result over the cache is
    merged with a partial over other keys by ``combine``, as a shared prefix would be."""
    D, H, Hkv, page = 128, 8, 2, 32
    prompts, steps = [45, 3, 70], 4
    s = Setup([p + steps for p in prompts], prompts, H=H, Hkv=Hkv, D=D, page=page, rot=D, seed=21,
              dtype=torch.float16)
    want = s.pages()
    for step in range(steps + 1):
        new = prompts if step == 0 else [1, 1, 1]
        lens = [p + step for p in prompts]
        g = torch.Generator().manual_seed(50 + step)
        s.q, s.k, s.v = torch.randn(sum(new), H + 2 * Hkv, D, generator=g).half().cuda().split([H, Hkv, Hkv], 1)
        s.lens, s.new, s.cu = lens, new, [0, new[0], new[0] + new[1], sum(new)]
        s.lens_d.copy_(torch.tensor(lens))
        s.cu_d.copy_(torch.tensor(s.cu))
        q_want = ref.append(want, s.k, s.v, s.table.tolist(), lens, s.cu, q=s.q, cos=s.cos, sin=s.sin)
        s.q = s.append()
        assert torch.equal(s.q.cpu(), narrow(q_want, torch.float16))
        same_pages(s.pages(), want)
        check_attention(s)
    o, lse = s.attend()
    other = torch.randn(3, H, 1, D, generator=s.g).half().cuda()
    lse_b = torch.randn(3, H, 1, generator=s.g).cuda() + 3
    got, got_lse = fused_attn.combine([o[:, :, None], other], [lse[:, :, None], lse_b])
    w = torch.sigmoid(lse.double() - lse_b[:, :, 0].double())[..., None]
    expect = w * o.double() + (1 - w) * other[:, :, 0].double()
    # one rounding of the output and of the two inputs' weights in fp32
    assert bool(((got[:, :, 0].double() - expect).abs() <= 2.0**-11 * expect.abs() + 1e-6).all())
    assert torch.allclose(got_lse[:, :, 0].double(), torch.logaddexp(lse.double(), lse_b[:, :, 0].double()), atol=1e-5)


def test_other_stream_and_graph():
    s = Setup([90, 260], [1, 1], rot=128, seed=22, page=32)
    s.cos, s.sin = (torch.cat([t, t.flip(0)[:9]]) for t in (s.cos, s.sin))
    want = s.pages()
    q_want = ref.append(want, s.k, s.v, s.table.tolist(), s.lens, s.cu, q=s.q, cos=s.cos, sin=s.sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    with torch.cuda.stream(side):
        s.append()
        s.attend()
        pool = torch.cuda.graph_pool_handle()
        for g in graphs:  # two graphs that share their memory
            with torch.cuda.graph(g, stream=side, pool=pool):
                q = s.append()
                outs.append((q, *s.attend(q=q)))
    torch.cuda.current_stream().wait_stream(side)
    kept = s.q
    for g, (q, o, lse) in list(zip(graphs, outs)) * 2:
        g.replay()
        torch.cuda.synchronize()
        same_pages(s.pages(), want)
        assert torch.equal(q.cpu(), narrow(q_want, s.dtype))
        s.q = q
        check_attention(s, o=o, lse=lse)
        s.q = kept
    # a replay follows the lengths that the program wrote before it
    s.lens = [91, 261]
    s.lens_d.copy_(torch.tensor(s.lens))
    q_want = ref.append(want, s.k, s.v, s.table.tolist(), s.lens, s.cu, q=s.q, cos=s.cos, sin=s.sin)
    graphs[1].replay()
    torch.cuda.synchronize()
    same_pages(s.pages(), want)
    q, o, lse = outs[1]
    assert torch.equal(q.cpu(), narrow(q_want, s.dtype))
    s.q = q
    check_attention(s, o=o, lse=lse)
    del graphs, outs


def test_bad_device_values_are_skipped_and_reported():
    """Pages, lengths, offsets and positions out of range: nothing is written outside, the rest of the
    batch is served, and the status says so."""
    def fresh():
        return Setup([20, 33], [4, 3], rot=128, seed=23)

    for what in ("page", "negative page", "length", "negative length", "offsets", "offset order", "angles"):
        s = fresh()
        good = fresh()
        if what in ("page", "negative page"):
            s.table_d[0, 1] = s.P if what == "page" else -1
        elif what == "length":
            s.lens_d[0] = 10**6
        elif what == "negative length":
            s.lens_d[0] = -5
        elif what == "offsets":
            s.cu_d[2] = 100
        elif what == "offset order":
            s.cu_d[0] = 5
        elif what == "angles":
            s.cos, s.sin = s.cos[:18].contiguous(), s.sin[:18].contiguous()
        q = s.append()
        torch.cuda.synchronize()
        assert fused_attn.last_device_error() == (1, 1 << 11), what
        o, lse = s.attend()
        torch.cuda.synchronize()
        if what != "angles":
            assert fused_attn.last_device_error() == (1, 1 << 11), what
        good.append()
        o_good, _ = good.attend()
        if what not in ("offsets", "offset order", "angles"):  # the second sequence is as it should be
            assert torch.equal(o[4:], o_good[4:]) or bool((o[4:] - o_good[4:]).abs().max() < 0.05)
        assert q.shape == s.q.shape and bool(torch.isfinite(o).all())
        spare = torch.ones(s.P, dtype=torch.bool)
        spare[[int(p) for row in s.table.tolist() for p in row if p >= 0]] = False
        for a, b in ((s.k_cache, fresh().k_cache), (s.v_cache, fresh().v_cache)):
            assert torch.equal(a.view(torch.uint8)[spare.cuda()], b.view(torch.uint8)[spare.cuda()])
        fused_attn.last_device_error()


@pytest.mark.parametrize("new", [[4, 3, 2], [40, 33, 50]])
@pytest.mark.parametrize("offset,value,skipped", [(0, 2, [0]), (1, -1, [0, 1]), (1, 10**6, [0, 1]), (3, 10**6, [2])])
def test_rows_of_sequences_with_bad_offsets_are_zero(new, offset, value, skipped):
    s = Setup([60, 70, 80], new, rot=128, seed=26)
    rows = sum(new)
    bounds = s.cu_d.tolist()
    s.cu_d[offset] = value
    garbage = torch.full((rows * s.H * s.D * 4,), float("nan"), device="cuda")  # what a reused block may hold
    del garbage
    q = s.append()
    o, lse = s.attend()
    torch.cuda.synchronize()
    assert fused_attn.last_device_error() == (1, 1 << 11)
    assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(lse).all())
    for i in range(len(new)):
        part = slice(bounds[i], bounds[i + 1])
        zero = i in skipped
        assert bool((o[part] == 0).all()) == zero and bool((lse[part] == 0).all()) == zero
        assert bool((q[part] == 0).all()) == zero


def test_refusals_of_the_op():
    s = Setup([20, 33], [4, 3], rot=128, seed=24)
    args = dict(k=s.k, v=s.v, k_cache=s.k_cache, v_cache=s.v_cache, k_scale=s.k_scale, v_scale=s.v_scale,
                block_table=s.table_d, seq_lens=s.lens_d, cu_seqlens=s.cu_d, q=s.q, cos=s.cos, sin=s.sin)

    def refuse(match, **change):
        with pytest.raises(RuntimeError, match=match):
            fused_attn.cache_append(**{**args, **change})

    refuse("float16 or bfloat16", k=s.k.float())
    refuse("of one dtype", v=s.v.half())
    refuse("float8_e4m3fn", k_cache=s.k_cache.view(torch.uint8))
    refuse("contiguous float32", k_scale=s.k_scale.half())
    refuse("contiguous float32", v_scale=s.v_scale[:-1])
    refuse("int32", block_table=s.table_d.long())
    refuse("int32", seq_lens=s.lens_d.long())
    refuse("cu_seqlens must be", cu_seqlens=s.cu_d[:-1])
    refuse("must be a multiple", cu_seqlens=None, k=s.k[:5], v=s.v[:5], q=s.q[:5])
    refuse("come together", sin=None)
    refuse("needs cos and sin", cos=None, sin=None)
    refuse("rot_dim", cos=s.cos[:, :12].contiguous(), sin=s.sin[:, :12].contiguous())
    refuse("contiguous, 16-byte", cos=s.cos[:, ::2], sin=s.sin[:, ::2])
    refuse("multiples of 16 bytes", k=s.k[:, :1].expand(-1, 2, -1))
    refuse("heads", k=s.k[..., :64], v=s.v[..., :64])
    refuse("cache's device", seq_lens=s.lens_d.cpu())
    refuse("page_size", k_cache=s.k_cache[:, :, :8], v_cache=s.v_cache[:, :, :8])
    with pytest.raises(RuntimeError, match="multiple of Hkv"):
        fused_attn.cache_attention(s.q[:, :3], s.k_cache, s.v_cache, s.k_scale, s.v_scale, s.table_d, s.lens_d,
                                   cu_seqlens=s.cu_d)
    with pytest.raises(RuntimeError, match="scale must be"):
        s.attend(scale=-1.0)
    assert fused_attn.last_device_error() == (0, 0)


def test_empty_calls():
    s = Setup([20, 33], [0, 0], rot=128, seed=25)
    before = s.pages()
    q = s.append()
    o, lse = s.attend()
    assert q.shape == (0, 4, 128) and o.shape == (0, 4, 128) and lse.shape == (0, 4)
    same_pages(s.pages(), before)
    s = Setup([20], [0], rot=128, seed=25, tail=5)
    before = s.pages()
    assert not bool(s.append().any())
    o, lse = s.attend()
    assert not bool(o.any()) and not bool(lse.any())
    same_pages(s.pages(), before)


def test_pages_past_two_gigabytes():
    """Offsets that pass 32 bits: the batch's pages are the last ones of a pool of 2.4 GB."""
    D, Hkv, page, P = 128, 8, 128, 18500
    assert P * Hkv * page * D > 2**31
    k_cache = torch.zeros(P, Hkv, page, D, dtype=E4M3, device="cuda")
    v_cache = torch.zeros(P, Hkv, page, D, dtype=E4M3, device="cuda")
    small = Setup([200, 130], [200, 1], H=8, Hkv=Hkv, page=page, rot=D, seed=26)
    n = small.P
    shift = P - n
    k_cache[shift:], v_cache[shift:] = small.k_cache, small.v_cache
    scales = [torch.ones(P, Hkv, device="cuda") for _ in range(2)]
    scales[0][shift:], scales[1][shift:] = small.k_scale, small.v_scale
    table = torch.where(small.table_d >= 0, small.table_d + shift, small.table_d)
    args = dict(block_table=table, seq_lens=small.lens_d, cu_seqlens=small.cu_d)
    q = fused_attn.cache_append(small.k, small.v, k_cache, v_cache, *scales, q=small.q, cos=small.cos,
                                sin=small.sin, **args)
    o, lse = fused_attn.cache_attention(q, k_cache, v_cache, *scales, return_lse=True, **args)
    q2 = small.append()
    o2, lse2 = small.attend(q=q2)
    assert torch.equal(q, q2) and torch.equal(o, o2) and torch.equal(lse, lse2)
    assert torch.equal(k_cache[shift:].view(torch.uint8), small.k_cache.view(torch.uint8))
    assert not bool(k_cache[:shift].view(torch.uint8).any())
    assert fused_attn.last_device_error() == (0, 0)


def test_opcheck():
    """Fake kernels against the real ones (the schema check cannot compare float8 tensors)."""
    s = Setup([20, 33], [4, 3], rot=128, seed=27)
    tail = (s.k_cache, s.v_cache, s.k_scale, s.v_scale, s.table_d, s.lens_d, s.cu_d)
    ops = torch.ops.fused_attn
    torch.library.opcheck(ops.cache_attention, (s.q, *tail, True, 0.1), test_utils="test_faketensor")
    torch.library.opcheck(ops.cache_append, (s.q, s.k, s.v, *tail, s.cos, s.sin, False),
                          test_utils="test_faketensor")
