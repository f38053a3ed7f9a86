"""The paged 8-bit cache without a GPU: the oracle's own properties, refusals of the C ABI before a
device is looked at, schemas and fake kernels."""

from __future__ import annotations

import math

import pytest
import torch

import fused_attn
from fused_attn import abi
from oracle import cache as ref

needs_lib = pytest.mark.skipif(not abi.available(), reason="libfa_sm100.so not built")
needs_ext = pytest.mark.skipif(not fused_attn.is_available(), reason="fused_attn._C not built")


# ---- the oracle ----


def test_magnitudes_are_the_formats():
    got = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    assert torch.equal(got, ref.MAGNITUDES)


def test_round_e4m3_equals_the_types_own_rounding():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20000, generator=g) * torch.exp(3 * torch.randn(20000, generator=g))
    x = torch.cat([x.clamp(-448, 448), torch.tensor([0.0, 2.0**-10, 3 * 2.0**-10, 17.0, 19.0])])
    assert torch.equal(ref.round_e4m3(x), x.to(torch.float8_e4m3fn).float().double())


@pytest.mark.parametrize("amax,exp", [(448.0, 0), (448.0000001, 1), (447.9, 0), (224.0, -1), (1.75, -8),
                                      (0.0, -64), (1e-30, -64), (3.4e38, 120)])
def test_needed_exp(amax, exp):
    assert ref.needed_exp(amax) == exp


def test_append_in_steps_keeps_earlier_rows_on_the_pages_step():
    """One row at a time: a page's scale never falls, and what is stored stays within one rounding
    (2^-4 relative, half the least step absolute) of the value for each time the scale grew."""
    g = torch.Generator().manual_seed(2)
    c = ref.Pages(*(torch.zeros(2, 1, 16, 64, dtype=torch.float64) for _ in range(2)),
                  *(torch.ones(2, 1, dtype=torch.float64) for _ in range(2)))
    rows = torch.randn(20, 1, 64, generator=g) * torch.logspace(-3, 2, 20)[:, None, None]
    last = 0.0
    for i in range(20):
        ref.append(c, rows[i:i + 1], rows[i:i + 1], [[1, 0]], [i + 1])
        scale = float(c.k_scale[1 if i < 16 else 0, 0])
        assert i == 16 or scale >= last
        last = scale
    got = torch.cat([c.k[1, 0] * c.k_scale[1, 0], c.k[0, 0, :4] * c.k_scale[0, 0]])
    step = torch.cat([c.k_scale[1, 0].expand(16), c.k_scale[0, 0].expand(4)])[:, None] * 2.0**-9
    err = (got - rows[:, 0].double()).abs()
    assert bool((err <= rows[:, 0].double().abs() * 2.0**-4 + 16 * step / 2).all())


def test_attention_of_the_oracle_is_softmax():
    g = torch.Generator().manual_seed(3)
    c = ref.Pages(*(ref.round_e4m3(torch.randn(3, 2, 16, 64, generator=g)) for _ in range(2)),
                  *(torch.tensor([[1.0, 2.0], [0.5, 0.25], [4.0, 1.0]], dtype=torch.float64)
                    for _ in range(2)))
    q = torch.randn(3, 4, 64, generator=g)
    got = ref.attention(c, q, [[2, 0]], [21])
    k = torch.cat([c.k[2] * c.k_scale[2][:, None, None], c.k[0] * c.k_scale[0][:, None, None]], 1)
    v = torch.cat([c.v[2] * c.v_scale[2][:, None, None], c.v[0] * c.v_scale[0][:, None, None]], 1)
    for i in range(3):
        for x in range(4):
            a = (k[x // 2, :19 + i] @ q[i, x].double()) / 8
            p = torch.softmax(a, 0)
            assert torch.allclose(got.o[i, x], p @ v[x // 2, :19 + i], rtol=1e-12, atol=1e-13)
            assert math.isclose(float(got.lse[i, x]), float(torch.logsumexp(a, 0)), rel_tol=1e-12)
    empty = ref.attention(c, q, [[2, 0]], [2])  # the first of three queries sees nothing
    assert float(empty.lse[0, 0]) == math.inf and not bool(empty.o[0].any())


# ---- refusals of the C ABI: fake addresses, rejected before they are used ----

P16 = 0x1000


def a_cache(**change) -> abi.FaCache:
    c = abi.FaCache(P16, P16, P16, P16, 8, 16, 2, 128, (4096, 2048, 128), (4096, 2048, 128), P16, 4, 4,
                    P16, None, 3)
    for name, value in change.items():
        if name.endswith("strides"):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


def a_step(**change) -> abi.FaAppend:
    p = abi.FaAppend(P16, P16, (256, 128), (256, 128), P16, P16, (512, 128), 4, P16, P16, 64, 128, 0)
    for name, value in change.items():
        if name.endswith("strides"):
            getattr(p, name)[:] = value
        else:
            setattr(p, name, value)
    return p


BAD_CACHES = [dict(D=96), dict(page_size=8), dict(page_size=48), dict(page_size=256), dict(Hkv=0), dict(num_pages=0),
              dict(n_seqs=0), dict(max_pages=0), dict(table_stride=3), dict(k=None), dict(v=P16 + 8),
              dict(k_scale=None), dict(v_scale=P16 + 2), dict(block_table=None), dict(seq_lens=None),
              dict(seq_lens=P16 + 1), dict(cu_seqlens=P16 + 2), dict(k_strides=(4096, 2048, 120)),
              dict(v_strides=(0, 2048, 128)), dict(k_strides=(4096, -2048, 128)),
              dict(max_pages=1 << 28, table_stride=1 << 28)]


@needs_lib
@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(bad):
    c = a_cache(**bad)
    assert abi.cache_append(1, c, a_step(), 3) == abi.CUDA_ERROR_INVALID_VALUE
    assert abi.cache_attention(1, c, P16, (512, 128), P16, P16, P16, 3, 4, 0.1, True) == \
        abi.CUDA_ERROR_INVALID_VALUE
    assert abi.cache_attention_workspace_bytes(c, 4, 3) == 0


@needs_lib
@pytest.mark.parametrize("bad", [dict(k=None), dict(v=P16 + 8), dict(k_strides=(256, 4)), dict(v_strides=(0, 128)),
                                 dict(cos=None), dict(sin=P16 + 4), dict(rot_dim=24), dict(rot_dim=144),
                                 dict(rot_dim=0), dict(table_rows=0), dict(H=0), dict(q_out=None), dict(q=P16 + 2),
                                 dict(q_strides=(512, 127)), dict(cos=None, sin=None)], ids=str)
def test_bad_steps_are_refused(bad):
    assert abi.cache_append(1, a_cache(), a_step(**bad), 3) == abi.CUDA_ERROR_INVALID_VALUE


@needs_lib
def test_other_refusals():
    c, p = a_cache(), a_step()
    bad = abi.CUDA_ERROR_INVALID_VALUE
    assert abi.cache_append(0, c, p, 3) == bad  # fp32
    assert abi.cache_append(1, None, p, 3) == bad and abi.cache_append(1, c, None, 3) == bad
    assert abi.cache_append(1, c, p, 4) == bad  # 4 tokens, 3 sequences, no offsets
    assert abi.cache_append(1, c, p, -3) == bad

    def attend(dtype=1, q=P16, strides=(512, 128), o=P16, lse=P16, ws=P16, T=3, H=4, scale=0.1):
        return abi.cache_attention(dtype, c, q, strides, o, lse, ws, T, H, scale, True)

    assert attend(dtype=0) == bad and attend(H=3) == bad and attend(H=0) == bad
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert attend(scale=scale) == bad
    assert attend(q=0) == bad and attend(o=P16 + 8) == bad and attend(lse=0) == bad
    assert attend(strides=(512, 100)) == bad and attend(T=2) == bad
    assert abi.cache_attention_workspace_bytes(c, 3, 3) == 0
    assert abi.cache_attention_workspace_bytes(c, 4, 3) > 0


# ---- the op surface ----


@needs_ext
def test_schemas_name_what_is_written():
    s = str(torch.ops.fused_attn.cache_append.default._schema)
    assert "Tensor(a!) k_cache" in s and "Tensor(d!) v_scale" in s and s.endswith("-> Tensor")
    assert str(torch.ops.fused_attn.cache_attention.default._schema).endswith("-> (Tensor, Tensor)")


@needs_ext
def test_fakes_give_metadata():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def e(*shape, dtype=torch.float16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        pool = e(9, 2, 16, 64, dtype=torch.float8_e4m3fn)
        sc = e(9, 2, dtype=torch.float32)
        table, lens = e(3, 4, dtype=torch.int32), e(3, dtype=torch.int32)
        q, k = e(6, 4, 64), e(6, 2, 64)
        cos = e(100, 32, dtype=torch.float32)
        o, lse = fused_attn.cache_attention(q, pool, pool, sc, sc, table, lens, return_lse=True)
        assert o.shape == q.shape and o.dtype == q.dtype
        assert tuple(lse.shape) == (6, 4) and lse.dtype == torch.float32
        turned = fused_attn.cache_append(k, k, pool, pool, sc, sc, table, lens, q=q, cos=cos, sin=cos)
        assert turned.shape == q.shape and turned.is_contiguous()
        assert fused_attn.cache_append(k, k, pool, pool, sc, sc, table, lens) is None
        with pytest.raises(RuntimeError, match="needs cos and sin"):
            fused_attn.cache_append(k, k, pool, pool, sc, sc, table, lens, q=q)
        with pytest.raises(RuntimeError, match="float8_e4m3fn"):
            fused_attn.cache_attention(q, q[None], q[None], sc, sc, table, lens)
        with pytest.raises(RuntimeError, match="D must be 64 or 128"):
            bad = e(9, 2, 16, 96, dtype=torch.float8_e4m3fn)
            fused_attn.cache_attention(q, bad, bad, sc, sc, table, lens)
