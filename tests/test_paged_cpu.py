"""The paged cache's argument checks, which come before anything reaches the library, and its plain counterpart's own arithmetic."""
import math

import pytest
import torch

from sharpmind_b200 import ops, paged
from tests import paged_util


class _Lib:
    """Stands in for the library: no call may reach it."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


class _Ctx:
    device, h, lib = 0, None, _Lib()


def _cache(pages=4, kvh=2, page=16, dim=64):
    """A cache as the constructor leaves it, on the CPU (the constructor itself refuses that)."""
    c = object.__new__(paged.PagedKVCache)
    c.torch, c.ctx, c.device = torch, _Ctx(), torch.device("cpu")
    c.pages, c.kv_heads, c.page, c.head_dim = pages, kvh, page, dim
    c._types, c._index, c._kv_ref = {torch.float32: 0, torch.bfloat16: 30}, -1, None  # (-1: the CPU)
    return c


def _codes(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


@pytest.mark.parametrize("k,v,scales,error,text", [
    (_codes(4, 2, 16, 64), _codes(4, 2, 64, 16), torch.zeros(4, 2, 2), ops.ArgumentException, "context's device"),
    (_codes(4, 2, 48, 64), _codes(4, 2, 64, 48), torch.zeros(4, 2, 2), ops.NotSupportedException, "48"),
    (_codes(4, 2, 16, 96), _codes(4, 2, 96, 16), torch.zeros(4, 2, 2), ops.NotSupportedException, "96"),
    (_codes(4, 2, 16, 64), _codes(4, 2, 16, 64), torch.zeros(4, 2, 2), ops.ArgumentException, "values are"),
    (_codes(4, 2, 16, 64), _codes(4, 2, 64, 16), torch.zeros(4, 2), ops.ArgumentException, "scales are"),
    (torch.zeros(4, 2, 16, 64), _codes(4, 2, 64, 16), torch.zeros(4, 2, 2), ops.ArgumentException, "float8"),
    (_codes(4, 2, 16, 128)[..., ::2], _codes(4, 2, 64, 16), torch.zeros(4, 2, 2), ops.ArgumentException, "contiguous"),
    (_codes(4, 32, 64), _codes(4, 2, 64, 16), torch.zeros(4, 2, 2), ops.ArgumentException, "four"),
])
def test_the_constructor_refuses(k, v, scales, error, text):
    with pytest.raises(error, match=text):
        paged.PagedKVCache(_Ctx(), k, v, scales)


def _i(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_update_refuses():
    c, table, lens = _cache(), torch.zeros((2, 3), dtype=torch.int32), _i(5, 6)
    k, q = torch.zeros(2, 2, 64), torch.zeros(2, 4, 64)
    cos = torch.zeros(48, 32)
    bad = [
        (dict(k=k.half(), v=k.half()), ops.NotSupportedException, "float16"),
        (dict(v=k.bfloat16()), ops.ArgumentException, "v is of another"),
        (dict(k=torch.zeros(2, 3, 64)), ops.ArgumentException, "k is"),
        (dict(k=torch.zeros(2, 2, 128)[..., ::2], v=k), ops.ArgumentException, "contiguous"),
        (dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64)), ops.ArgumentException, "3 rows for 2"),
        (dict(lengths=_i(5)), ops.ArgumentException, "lengths"),
        (dict(lengths=torch.tensor([5, 6])), ops.ArgumentException, "lengths"),
        (dict(table=table.long()), ops.ArgumentException, "table"),
        (dict(table=torch.zeros((3, 2), dtype=torch.int32).T), ops.ArgumentException, "table"),
        (dict(row_start=_i(0, 2)), ops.ArgumentException, "row_start"),
        (dict(cos=cos), ops.ArgumentException, "together"),
        (dict(cos=cos, sin=cos[:3]), ops.ArgumentException, "cos and sin"),
        (dict(cos=cos.double(), sin=cos.double()), ops.ArgumentException, "cos and sin"),
        (dict(cos=torch.zeros(48, 30), sin=torch.zeros(48, 30)), ops.ArgumentException, "multiple of 8"),
        (dict(cos=torch.zeros(48, 40), sin=torch.zeros(48, 40)), ops.ArgumentException, "80 of 64"),
        (dict(q=q.bfloat16()), ops.ArgumentException, "q is of another"),
        (dict(q=q[:1]), ops.ArgumentException, "q is of another"),
        (dict(q=q, q_out=q[:, :2]), ops.ArgumentException, "q_out"),
        (dict(q=torch.zeros(2, 6, 64)[:, :4], q_out=torch.zeros(2, 4, 64)[:1]), ops.ArgumentException, "q_out"),
    ]
    for change, error, text in bad:
        with pytest.raises(error, match=text):
            c.Update(**{**dict(k=k, v=k, table=table, lengths=lens), **change})


def test_attention_and_read_refuse():
    c, table, lens, q = _cache(), torch.zeros((2, 3), dtype=torch.int32), _i(5, 6), torch.zeros(2, 4, 64)
    bad = [
        (dict(q=q.half()), ops.NotSupportedException, "float16"),
        (dict(q=q[:, :3]), ops.ArgumentException, "3 query heads on 2"),
        (dict(q=torch.zeros(2, 4, 32)), ops.ArgumentException, "q is"),
        (dict(q=torch.zeros(2, 8, 64)[:, ::2]), ops.ArgumentException, "contiguous"),
        (dict(out=q.bfloat16()), ops.ArgumentException, "out is"),
        (dict(out=torch.zeros(4, 2, 64).transpose(0, 1)), ops.ArgumentException, "out is"),
        (dict(lengths=_i(1, 2, 3)), ops.ArgumentException, "lengths"),
    ]
    for change, error, text in bad:
        with pytest.raises(error, match=text):
            c.attention(**{**dict(q=q, table=table, lengths=lens, scale=0.1), **change})
    with pytest.raises(ops.ArgumentException, match="pages"):
        c.read(torch.tensor([1]))
    with pytest.raises(ops.NotSupportedException):
        c.read(_i(1), torch.float16)


def test_the_library_refuses_without_a_context():
    """Null pointers and unknown sizes end in a status, not in a crash."""
    import ctypes as C

    from sharpmind_b200 import _lib

    lib, kv, sq = _lib.load(), paged._Kv(), paged._Seqs()
    assert lib.smc_paged_attention_work(None, C.byref(kv), 1, 1, 4, 1, 10) == -1
    assert lib.smc_paged_attention_work(None, None, 1, 1, 4, 1, 10) == -1
    assert lib.smc_paged_attention_dev(None, C.byref(kv), C.byref(sq), 0, None, 0, None, 4, 0.1, 0, 1, 10, None, 0, None) == 1
    assert lib.smc_paged_update_dev(None, C.byref(kv), C.byref(sq), 0, None, 0, None, 0, None, 0, None, 0, None, None, 0, 0, 0, None) == 1
    assert lib.smc_paged_read_dev(None, C.byref(kv), None, 1, 0, None, None, None) == 1


# ---- the plain counterpart
def test_plain_scales_and_codes():
    assert paged_util.exponent(0.0) == -40 and paged_util.exponent(448.0) == 0 and paged_util.exponent(448.1) == 1 and paged_util.exponent(224.0) == -1
    p = paged_util.PlainPages(2, 1, 16, 64)
    x = torch.randn(10, 1, 64, generator=torch.Generator().manual_seed(1))
    p.update(x, 5 * x, [[1]], [10], [10])
    k, v = p.values(1)
    # half a step of a four-bit number, or of the smallest code
    assert bool(((k[:10] - x).abs() <= (2.0 ** -4 * x.abs()).clamp(min=2.0 ** -10 * float(p.scales[1, 0, 0]))).all())
    assert bool(((v[:10] - 5 * x).abs() <= (2.0 ** -4 * 5 * x.abs()).clamp(min=2.0 ** -10 * float(p.scales[1, 0, 1]))).all())
    big = torch.full((1, 1, 64), 1000.0)
    p.update(big, big, [[1]], [11], [1])
    assert float(p.scales[1, 0, 0]) == 4.0
    k2, _ = p.values(1)
    # a larger scale changes only what falls below its normal codes
    large = k[:10].abs() >= 2.0 ** -6 * 4
    assert torch.equal(k2[:10][large], k[:10][large]) and bool(((k2[:10] - k[:10]).abs() <= 2.0 ** -10 * 4).all())


def test_plain_attention_is_the_softmax():
    p = paged_util.PlainPages(4, 1, 16, 64)
    x = torch.randn(40, 1, 64, generator=torch.Generator().manual_seed(2))
    p.update(x, x + 1, [[2, 0, 3]], [40], [40])
    q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(3))
    out, bound = paged_util.attention(p, q, [[2, 0, 3]], [40], [3], 0.125)
    k, v = p.tokens([2, 0, 3], 40)
    want = torch.softmax(q[1, 1].double() @ k[:39, 0].T * 0.125, 0) @ v[:39, 0]
    assert torch.allclose(out[1, 1], want, atol=1e-12) and float(bound.max()) < 1e-3
    out, _ = paged_util.attention(p, q, [[2, 0, 3]], [40], [3], 0.125, window=1)
    assert torch.allclose(out[:, 0], v[37:40, 0], atol=1e-12)
    assert math.isclose(float(paged_util.attention(p, q, [[2, 0, 3]], [0], [1], 0.125)[0].abs().max()), 0.0)
