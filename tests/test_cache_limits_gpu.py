"""The paged 8-bit cache at the ends of what its documents allow, against the 64-bit oracle (oracle/cache.py)."""

from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import fused_attn
from fused_attn import abi
from oracle import cache as ref
from test_cache_gpu import E4M3, Setup, check_append, check_attention, narrow, same_pages

pytestmark = pytest.mark.gpu

BAD_INDEX = (1, 1 << 11)


@pytest.fixture(autouse=True)
def _available():
    if not fused_attn.is_available() or not fused_attn.impl_supports(5, torch.float16, 128):
        pytest.skip("kernels not available")
    fused_attn.last_device_error()
    yield


def c_cache(s: Setup) -> abi.FaCache:
    P, Hkv, page, D = s.k_cache.shape
    strides = [tuple(c.stride(i) for i in range(3)) for c in (s.k_cache, s.v_cache)]
    return abi.FaCache(s.k_cache.data_ptr(), s.v_cache.data_ptr(), s.k_scale.data_ptr(), s.v_scale.data_ptr(), P,
                       page, Hkv, D, *strides, s.table_d.data_ptr(), s.table_d.stride(0), s.table_d.shape[1],
                       s.lens_d.data_ptr(), s.cu_d.data_ptr(), len(s.lens))


def attend_into_nan(s: Setup, causal=True):
    """The C entry point on outputs and a workspace that hold NaN: what is not written shows."""
    c = c_cache(s)
    T = s.q.shape[0]
    o = torch.full((T, s.H, s.D), math.nan, dtype=s.dtype, device="cuda")
    lse = torch.full((T, s.H), math.nan, device="cuda")
    ws = torch.full((abi.cache_attention_workspace_bytes(c, s.H, T),), 0xFF, dtype=torch.uint8, device="cuda")
    err = abi.cache_attention(abi.dtype_code(s.dtype), c, s.q.data_ptr(), (s.q.stride(0), s.q.stride(1)), o.data_ptr(),
                              lse.data_ptr(), ws.data_ptr(), T, s.H, 1 / math.sqrt(s.D), causal,
                              torch.cuda.current_stream().cuda_stream)
    assert err == 0
    torch.cuda.synchronize()
    return o, lse


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("H,Hkv,D,page,lens,new", [
    (8, 2, 128, 64, [64], [300]), (1, 1, 64, 128, [128], [1000]), (1, 1, 64, 128, [100], [300]),
    (6, 2, 64, 16, [16, 3, 0], [500, 90, 200]), (7, 1, 128, 32, [129, 250], [300, 250]), (300, 1, 64, 16, [5], [9])],
    ids=str)
def test_more_queries_than_keys(H, Hkv, D, page, lens, new, causal):
    """Many new tokens over a table with room for few keys: every row is written, those in front of the keys too."""
    s = Setup(lens, new, H=H, Hkv=Hkv, D=D, page=page, seed=61)
    o, lse = attend_into_nan(s, causal)
    check_attention(s, causal, o=o, lse=lse)


def test_a_length_above_the_tables_room_with_many_rows():
    """It counts as the room, and every row is written."""
    s = Setup([64, 40], [300, 30], H=4, Hkv=1, D=64, page=64, seed=62)
    s.lens_d[0] = 10**6
    o, lse = attend_into_nan(s)
    assert fused_attn.last_device_error() == BAD_INDEX
    check_attention(s, o=o, lse=lse)


@pytest.mark.parametrize("new", [1, 40], ids=["token", "rows"])
@pytest.mark.parametrize("low,high", [(-64, -64), (120, 120), (-64, 32), (24, 120)])
def test_value_scales_at_the_ends_of_their_range(low, high, new):
    """2^-64 and 2^120, alone and in one sequence with scales 2^96 away.

    The room grows with the scales' exponents: a score in units of log2 holds the exponent e, so it and the logarithm
    of the sum are rounded to half a step below 2^7, 2^-18 each, and P with them: 2^-17 of what P's own rounding to
    fp16, 2^-11, is in the oracle's room.  (The spread of 2^96 leaves 2^30 of the exponent's range for the scores.)"""
    s = Setup([200, 90], [new, new], seed=63)
    for at in range(s.P):
        s.v_scale[at] = 2.0 ** (high if at % 2 else low)
    o, lse = s.attend()
    want = ref.attention(s.pages(), s.q, s.table.tolist(), s.lens, s.cu)
    half = torch.finfo(s.dtype).eps / 2
    room = want.o_room * (1 + 2.0**-6) * (1 + half) + want.o.abs() * half
    assert bool(((o.cpu().double() - want.o).abs() <= room).all())
    assert bool(((lse.cpu().double() - want.lse).abs() <= want.lse_room + 2.0**-17).all())
    assert fused_attn.last_device_error() == (0, 0)


@pytest.mark.parametrize("new", [1, 40], ids=["token", "rows"])
@pytest.mark.parametrize("scale,end", [(1e-20, 2.0**-64), (0.0, 2.0**-64), (-1.0, 2.0**-64), (2.0**-140, 2.0**-64),
                                       (2.0**121, 2.0**120), (math.inf, 2.0**120)])
def test_value_scales_outside_their_range_are_reported(scale, end, new):
    """They count as the nearest end, and the status says so."""
    s = Setup([70, 90], [new, new], seed=64)
    s.v_scale[s.table[0, 1].item()] = end
    want = s.attend()
    assert fused_attn.last_device_error() == (0, 0)
    s.v_scale[s.table[0, 1].item()] = scale
    got = s.attend()
    assert fused_attn.last_device_error() == BAD_INDEX
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    s.v_scale[s.table[0, 1].item()] = end
    s.v_scale[[p for p in range(s.P) if p not in s.table.flatten().tolist()]] = scale  # a page that nobody has
    s.attend()
    assert fused_attn.last_device_error() == (0, 0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("lens,new,page,at", [([50, 40], [1, 1], 16, 1), ([50, 40], [20, 3], 16, 2),
                                              ([50, 40], [8, 3], 16, 3), ([100, 90], [60, 40], 16, 5),
                                              ([100, 90], [60, 40], 16, 6), ([700, 64], [300, 40], 128, 4)], ids=str)
def test_a_scale_that_is_nan_reaches_the_rows_that_see_its_page(lens, new, page, at, which, D):
    s = Setup(lens, new, page=page, D=D, seed=65)
    want = ref.attention(s.pages(), s.q, s.table.tolist(), s.lens, s.cu)
    (s.k_scale if which == "k" else s.v_scale)[s.table[0, at].item(), 1] = math.nan
    o, lse = s.attend()
    sees = torch.zeros(sum(new), s.H, dtype=torch.bool)
    for i in range(new[0]):
        sees[i, s.H // 2:] = lens[0] - new[0] + i >= at * page
    o, lse = o.cpu().double(), lse.cpu().double()
    assert torch.equal(torch.isnan(lse), sees)
    assert torch.equal(torch.isnan(o), sees[..., None].expand_as(o))
    half = torch.finfo(s.dtype).eps / 2
    room = want.o_room * (1 + half) + want.o.abs() * half
    assert bool(((lse - want.lse).abs() <= want.lse_room)[~sees].all())
    assert bool(((o - want.o).abs() <= room)[~sees].all())
    assert fused_attn.last_device_error() == (0, 0)


@pytest.mark.parametrize("n", [1, 3, 40], ids=["token", "draft", "rows"])
@pytest.mark.parametrize("over", [1, 2, 25, 10**6])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("rot", [None, 128], ids=["plain", "turned"])
def test_tokens_past_the_table_are_not_stored(n, over, page, rot):
    """A sequence that outgrows its table: the tokens that fit are stored, no row that was there changes, and the
    status says so."""
    s = Setup([128, 70], [n, 3], page=page, seed=66, rot=rot)
    s.lens[0] += over
    s.lens_d[0] += over
    if rot and over < 100:  # angles for all of the positions
        s.cos, s.sin = (torch.cat([t, t.flip(0)[:over]]) for t in (s.cos, s.sin))
    check_append(s, errors=BAD_INDEX)


@pytest.mark.parametrize("n", [1, 40], ids=["token", "rows"])
def test_the_largest_length_that_an_int_holds(n):
    """Its tokens have neither a page nor angles; the other sequence is stored."""
    s = Setup([70, 128], [30, n], page=32, seed=80, rot=128)
    s.lens[1] = 2**31 - 1
    s.lens_d[1] = 2**31 - 1
    check_append(s, errors=BAD_INDEX)
    _, lse = s.attend()
    assert fused_attn.last_device_error() == BAD_INDEX and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("S,at,value", [(4, 4, 2), (4, 4, 0), (4, 4, -1), (4, 4, 10**6), (4, 3, -1), (4, 3, 10**6),
                                        (4, 2, -5), (30, 17, -1), (30, 17, 10**6), (45, 45, 3), (45, 45, -1)])
def test_an_offset_out_of_range_costs_its_sequences_only(S, at, value):
    """The two sequences that an offset bounds store nothing and get zeros; the others are served."""
    new = [2 + i % 4 for i in range(S)]
    lens = [20 + 7 * i % 50 for i in range(S)]
    s, good = (Setup(lens, new, rot=128, seed=67) for _ in range(2))
    want = s.pages()
    s.cu_d[at] = value
    q = s.append()
    o, lse = s.attend(q=q)
    torch.cuda.synchronize()
    assert fused_attn.last_device_error() == BAD_INDEX
    for i in range(S):
        rows = slice(good.cu[i], good.cu[i + 1])
        if i in (at - 1, at):
            for x in (q, o, lse):
                assert not bool(x[rows].any())
            continue
        q_want = ref.append(want, s.k[rows], s.v[rows], [s.table[i].tolist()], [lens[i]], [0, new[i]], q=s.q[rows],
                            cos=s.cos, sin=s.sin)
        assert torch.equal(q[rows].cpu(), narrow(q_want, s.dtype))
    same_pages(s.pages(), want)
    q_good = good.append()
    o_good, lse_good = good.attend(q=q_good)
    for i in range(S):
        rows = slice(good.cu[i], good.cu[i + 1])
        if i not in (at - 1, at):
            assert bool(((lse[rows] - lse_good[rows]).abs() <= 1e-4).all())


@pytest.mark.parametrize("bounds", [[0, 50, 20, 60], [0, 100, 60, 20, 100], [0, 0, 90, 89, 100], [0, 30, 30, 0, 100]])
def test_offsets_that_descend_are_reported_by_append(bounds):
    """Every one in the batch, but some sequences end before they begin; pages of nobody stay as they are."""
    n = len(bounds) - 1
    s = Setup([120] * n, [25] * n, rot=128, seed=73, spare=5)
    assert s.q.shape[0] <= 100
    s.cu_d.copy_(torch.tensor(bounds).clamp(max=s.q.shape[0]))
    spare = torch.ones(s.P, dtype=torch.bool)
    spare[s.table.flatten().long()] = False
    before = s.k_cache.view(torch.uint8)[spare.cuda()].clone()
    s.append()
    torch.cuda.synchronize()
    assert fused_attn.last_device_error() == BAD_INDEX
    assert torch.equal(s.k_cache.view(torch.uint8)[spare.cuda()], before)


@pytest.mark.parametrize("scale", [17 / 18, 19 / 18, 17 / 22, 21 / 26, 0.7312847, 3.1415927, 1e-3])
@pytest.mark.parametrize("side", [-1, 0, 1])
def test_earlier_rows_under_a_scale_that_is_no_power_of_two_are_rounded_once(scale, side):
    """The scale next to a ratio that takes e4m3 values to the middle of two others, from below and above: the exact
    product of a value and such a ratio does not fit 24 bits, and its rounding to them would be a tie."""
    near = torch.tensor([scale], dtype=torch.float32)
    near = (near.view(torch.int32) + side).view(torch.float32).item()
    s = Setup([15], [1], seed=68, page=16)
    s.k_scale.fill_(near)
    s.v_scale.fill_(near * 2.0**30)
    for c in (s.k_cache, s.v_cache):
        every = torch.arange(s.P * 2 * 16 * 128, device="cuda").to(torch.uint8).view(s.P, 2, 16, 128)
        c.view(torch.uint8).copy_(every)
    check_append(s)


@pytest.mark.parametrize("new", [1, 70], ids=["token", "rows"])
def test_lengths_next_to_two_to_the_31(new):
    """One page under every entry of the longest table: no index wraps or is reported."""
    D, page = 64, 128
    entries = (2**31 - 1 - 128) // page
    g = torch.Generator(device="cuda").manual_seed(69)
    k, v = (torch.randn(2, 1, page, D, generator=g, device="cuda").to(E4M3) for _ in range(2))
    scales = [torch.ones(2, 1, device="cuda") for _ in range(2)]
    table = torch.ones(1, entries, dtype=torch.int32, device="cuda")
    lens = torch.tensor([entries * page], dtype=torch.int32, device="cuda")
    q = torch.randn(new, 1, D, generator=g, device="cuda").half()
    o, lse = fused_attn.cache_attention(q, k, v, *scales, table, lens, is_causal=False, return_lse=True)
    assert fused_attn.last_device_error() == (0, 0)
    _, one_lse = fused_attn.cache_attention(q, k, v, *scales, table[:, :1], lens.clamp(max=page), is_causal=False,
                                              return_lse=True)
    # A CTA's thread adds up to 2^31 / 128 / 148 / 2 tiles with 8 sums each in 32 bits, half a step each: 2^18.8 2^-24.
    assert bool(((lse - one_lse - math.log(entries)).abs() <= 2.0**-5).all()) and bool(torch.isfinite(o).all())


def test_outputs_and_pages_that_are_their_inputs_are_refused():
    """Blocks of one call would read what others write: one pool for keys and values, one tensor for q and o."""
    s = Setup([20, 33], [4, 3], rot=128, seed=74)
    kept = s.pages()
    with pytest.raises(RuntimeError, match="different tensors"):
        fused_attn.cache_append(s.k, s.v, s.k_cache, s.k_cache, s.k_scale, s.v_scale, s.table_d, s.lens_d, s.cu_d)
    with pytest.raises(RuntimeError, match="different tensors"):
        fused_attn.cache_append(s.k, s.v, s.k_cache, s.v_cache, s.k_scale, s.k_scale, s.table_d, s.lens_d, s.cu_d)
    c = c_cache(s)
    p = abi.FaAppend(s.k.data_ptr(), s.v.data_ptr(), (2 * 128, 128), (2 * 128, 128), s.q.data_ptr(), s.q.data_ptr(),
                     (4 * 128, 128), 4, s.cos.data_ptr(), s.sin.data_ptr(), s.cos.shape[0], 128, 0)
    T, code = s.q.shape[0], abi.dtype_code(s.dtype)
    assert abi.cache_append(code, c, p, T) == abi.CUDA_ERROR_INVALID_VALUE
    c.v = c.k
    p.q_out = torch.empty_like(s.q).data_ptr()
    assert abi.cache_append(code, c, p, T) == abi.CUDA_ERROR_INVALID_VALUE
    ws = torch.empty(abi.cache_attention_workspace_bytes(c, 4, T), dtype=torch.uint8, device="cuda")
    lse = torch.empty(T, 4, device="cuda")
    assert abi.cache_attention(code, c, s.q.data_ptr(), (4 * 128, 128), s.q.data_ptr(), lse.data_ptr(),
                               ws.data_ptr(), T, 4, 0.1, True) == abi.CUDA_ERROR_INVALID_VALUE
    same_pages(s.pages(), kept)
    # read only, one pool may hold both
    s.v_cache, s.v_scale = s.k_cache, s.k_scale
    check_attention(s)


@pytest.mark.parametrize("new", [1, 40], ids=["token", "rows"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_wait_that_runs_out_ends_the_call_with_a_status(D, new):
    """A limit of a nanosecond: the first wait that is not over at once runs out, with copies and products on their way.
    The kernels end by themselves, the host reads a timeout (or, where no wait was that long, has the result), and the
    next call is right."""
    s = Setup([3000, 500], [new, new], D=D, page=64, seed=75)
    s.attend()
    assert fused_attn.last_device_error() == (0, 0)
    fused_attn.set_wait_timeout_ns(1)
    try:
        o, lse = s.attend()
        err, bits = fused_attn.last_device_error()
    finally:
        fused_attn.set_wait_timeout_ns(2_000_000_000)
    assert err in (0, 702) and (bits != 0) == (err != 0)
    assert not bits & (1 << 7 | 1 << 11)  # neither a drain that gave up nor a bad index
    if err == 0:
        check_attention(s, o=o, lse=lse)
    check_attention(s)


@pytest.mark.parametrize("chunk", [200, 500])
def test_single_tokens_and_a_chunk_in_one_call(chunk):
    """A server's step: the batch's mean decides which kernel serves it, on both sides of the choice."""
    new = [1] * 40 + [chunk] + [1] * 23
    lens = [17 * i % 300 + 1 for i in range(64)]
    lens[40] = chunk + 333
    s = Setup(lens, new, H=4, Hkv=1, D=64, page=32, rot=64, seed=70)
    s.q = s.append()
    check_attention(s)


def test_a_step_under_torch_compile():
    """The ops' schemas and fakes carry a compiled step: pages and scales are changed in place."""
    s = Setup([90, 260], [3, 5], rot=128, seed=71, page=32)

    def step(q, k, v, k_cache, v_cache, k_scale, v_scale, table, lens, cu, cos, sin):
        q = fused_attn.cache_append(k, v, k_cache, v_cache, k_scale, v_scale, table, lens, cu, q=q, cos=cos, sin=sin)
        return q, *fused_attn.cache_attention(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, return_lse=True)

    want = s.pages()
    q_want = ref.append(want, s.k, s.v, s.table.tolist(), s.lens, s.cu, q=s.q, cos=s.cos, sin=s.sin)
    q, o, lse = torch.compile(step, backend="aot_eager", fullgraph=True)(
        s.q, s.k, s.v, s.k_cache, s.v_cache, s.k_scale, s.v_scale, s.table_d, s.lens_d, s.cu_d, s.cos, s.sin)
    same_pages(s.pages(), want)
    assert torch.equal(q.cpu(), narrow(q_want, s.dtype))
    s.q = q
    check_attention(s, o=o, lse=lse)


FIRST_CALL = """
import sys
import torch
sys.path[:0] = [{tests!r}, {root!r}, {package!r}]
import fused_attn
from test_cache_gpu import Setup, check_attention
for new, page in ((1, 32), (70, 32)):
    s = Setup([90, 260], [new, new], rot=128, seed=72, page=page)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = s.append()
        o, lse = s.attend(q=q)
    g.replay()
    torch.cuda.synchronize()
    s.q = q
    check_attention(s, o=o, lse=lse)
    del g
print("captured")
"""


def test_the_first_call_of_a_process_can_be_captured():
    tests = Path(__file__).resolve().parent
    code = FIRST_CALL.format(tests=str(tests), root=str(tests.parent),
                             package=str(tests.parent / "fused-attention-cuda_b200"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 40], ids=["token", "draft", "rows"])
def test_a_query_that_is_not_finite_stays_in_its_row(new, dtype):
    s = Setup([300, 77], [new, new], D=64, page=32, seed=76, dtype=dtype)
    want = ref.attention(s.pages(), s.q, s.table.tolist(), s.lens, s.cu)
    s.q[0, 1, 7] = math.nan
    s.q[new, 0, 3] = math.inf
    o, lse = s.attend()
    hit = torch.zeros(2 * new, s.H, dtype=torch.bool)
    hit[0, 1] = hit[new, 0] = True
    o, lse = o.cpu().double(), lse.cpu().double()
    assert bool(torch.isnan(o[hit]).all()) and bool(torch.isnan(lse[hit]).all())
    half = torch.finfo(dtype).eps / 2
    room = want.o_room * (1 + half) + want.o.abs() * half + 1e-7
    assert bool(((lse - want.lse).abs() <= want.lse_room)[~hit].all())
    assert bool(((o - want.o).abs() <= room)[~hit].all())


def test_calls_at_once_on_three_streams():
    """Both attention kernels, appends and the forward side by side: the bits of the calls made alone."""
    batches = [Setup([2000, 900], [300, 170], H=8, Hkv=2, page=64, rot=128, seed=77),
               Setup([1500, 40, 333], [1, 1, 1], H=8, Hkv=2, page=16, rot=128, seed=78),
               Setup([600] * 6, [600] * 6, H=4, Hkv=2, D=64, page=32, rot=64, seed=79, dtype=torch.float16)]
    x = torch.randn(2, 4, 512, 128, device="cuda").half()
    alone = []
    for s in batches:
        q = s.append()
        alone.append((q, *s.attend(q=q), fused_attn.forward(x, x, x)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[] for _ in batches]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for s, st, out in zip(batches, streams, got):
            with torch.cuda.stream(st):
                q = s.append()
                out.append((q, *s.attend(q=q), fused_attn.forward(x, x, x)))
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert fused_attn.last_device_error() == (0, 0)
