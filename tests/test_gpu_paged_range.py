"""Paged attention where value scales, or a row's weights, lie far apart.  The bound here is relative to what a row sums up, dimension by dimension, so that a
result which vanishes, or a sum that loses a key, is seen."""
import math

import pytest
import torch

from sharpmind_b200 import ops
from tests import paged_util
from tests.test_gpu_paged import Pair, gen, ints, near, randn, starts

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def tight(pages, q, table_row, length, scale, many):
    """(out, bound) in 64 bits for the last rows of one sequence.

    With p_j the softmax's weights, s_j the value scales and c_j the codes, out = sum p_j s_j c_j.  The weights p_j and their sum are off by the factor
    e^d (1 + 2^-21) each and sums of n by n 2^-23, as paged_util.attention derives, now of sum_j |p_j s_j c_j|: (4 d + n 2^-23 + 2^-19) of it.  Weights enter the
    second product as fp16: bfloat16 rounds them to 11 bits, another 2^-11; and none is held finer than 2^-25, where the largest p_j s_j stands for 2^14 at least (few
    rows) or 2^6 at least (many: the largest of a row's first 64 keys does, and a larger one later moves the reference up): 2^-39 or 2^-31 of the largest p_j s_j, times
    sum_j |c_j|.  bfloat16 results are rounded, 2^-8 |out|."""
    n, heads, dim = q.shape
    k, v = (x.cuda() for x in pages.tokens(table_row, length))
    ids = [int(x) for x in table_row[:-(-length // pages.page)]]
    s = pages.scales[ids, :, 1].repeat_interleave(pages.page, 0)[:length].double().cuda()  # [length, kvh]
    pos, j = torch.arange(length - n, length, device="cuda"), torch.arange(length, device="cuda")
    sees = j[None] <= pos[:, None]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for h in range(heads):
        g = h // (heads // pages.kvh)
        qq = q[:, h].double().cuda()
        p = torch.softmax((qq @ k[:, g].T * scale).masked_fill(~sees, -math.inf), -1)
        o, spread = p @ v[:, g], p @ v[:, g].abs()
        d = (2.0 ** -22 + dim * 2.0 ** -24) * (qq.abs() @ k[:, g].abs().T * scale).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
        codes = sees.double() @ (v[:, g].abs() / s[:, g:g + 1])
        b = (4 * d + length * 2.0 ** -23 + 2.0 ** -19) * spread + 2.0 ** (-31 if many else -39) * (p * s[:, g]).amax(-1, keepdim=True) * codes
        if q.dtype == BF16:
            b = b + 2.0 ** -11 * spread + 2.0 ** -8 * o.abs()
        out[:, h], bound[:, h] = o.cpu(), b.cpu()
    return out, bound


def put_codes(p, exponents, tag):
    """Codes of all magnitudes on both sides, keys of ordinary size; exponents: of the value scales, page after page of the first sequence."""
    p.plain.k[:] = torch.randint(0, 112, p.plain.k.shape, dtype=torch.uint8, generator=gen("codes", tag)) | (torch.randint(0, 2, p.plain.k.shape, dtype=torch.uint8, generator=gen("signs", tag)) << 7)
    p.plain.v[:] = torch.randint(0, 112, p.plain.v.shape, dtype=torch.uint8, generator=gen("vcodes", tag)) | (torch.randint(0, 2, p.plain.v.shape, dtype=torch.uint8, generator=gen("vsigns", tag)) << 7)
    p.plain.scales[:] = 2.0 ** -5
    for i, e in enumerate(exponents):
        p.plain.scales[int(p.table[0, i]), :, 1] = 2.0 ** e
    p.upload()


def is_many(rows, group, length):
    """The form that a call of one sequence takes: up to 16 pairs the one of a few rows, up to 64 where there are fifteen tiles of 64 keys for each 16 of them."""
    pairs = rows * group
    return not (pairs <= 16 or (pairs <= 64 and -(-length // 64) >= 15 * -(-pairs // 16)))


ORDERS = {
    "small first": lambda n: [-40] * (n // 2) + [108] * (n - n // 2),
    "large first": lambda n: [108] * (n // 2) + [-40] * (n - n // 2),
    "in turn": lambda n: [(-40, 119)[i % 2] for i in range(n)],
    "one large": lambda n: [119 if i == n // 3 else -30 for i in range(n)],
    "three kinds": lambda n: [(-40, 0, 100)[i % 3] for i in range(n)],
}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("rows,length,page", [(1, 450, 16), (1, 9000, 64), (4, 6000, 32), (16, 4500, 64), (40, 450, 16), (150, 1500, 32), (70, 6000, 64)])
def test_value_scales_far_apart_leave_the_sum_of_the_weights(cuda, dtype, order, rows, length, page):
    """Blocks of values 2^100 to 2^159 apart, within a unit of keys, between warps, runs and pieces: a key under a small scale counts in the softmax's sum like any other."""
    dim, heads = 64, 8
    p = Pair(cuda, [length], page=page, dim=dim, tag="scales")
    put_codes(p, ORDERS[order](p.width), (rows, length))
    q = (randn((rows, heads, dim), "q far", rows) * 0.05 * torch.exp2(torch.arange(heads) % 4).reshape(1, heads, 1)).to(dtype)
    got = p.cache.attention(q.cuda(), p.dtable, ints([length]), dim ** -0.5, row_start=starts([rows]), max_rows=rows, max_len=length).cpu().double()
    want, bound = tight(p.plain, q, p.table[0], length, dim ** -0.5, many=is_many(rows, heads // 2, length))
    off = (got - want).abs()
    assert bool(torch.isfinite(got).all()) and bool((off <= bound).all()), float((off / bound).max())
    assert cuda.device_status() == 0


def test_a_block_of_zeros_counts_beside_a_block_of_large_values(cuda):
    """Equal scores over as many zeros as values of 1e35: half of them."""
    p = Pair(cuda, [32], page=16, dim=64)
    k, v = torch.zeros((32, 2, 64)), torch.zeros((32, 2, 64))
    v[16:] = 1e35
    p.update([32], [32], k, v)
    p.same()
    for rows in (1, 30):
        q = torch.ones((rows, 4, 64))
        got = p.cache.attention(q.cuda(), p.dtable, ints([32]), 0.125, row_start=starts([rows]), max_rows=rows)
        value = float(p.plain.values(int(p.table[0, 1]))[1][0, 0, 0])
        assert torch.allclose(got[-1].cpu() / value, torch.full((4, 64), 0.5), rtol=2.0 ** -18, atol=0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,length", [(1, 450), (4, 6000), (16, 4500), (200, 450), (70, 3000)])
@pytest.mark.parametrize("ahead", [9.0, 14.0])
def test_a_first_key_that_takes_the_weight_and_has_no_value(cuda, dtype, rows, length, ahead):
    """The first key's score lies `ahead` above the others', its value is zero: what the rest sums up to is the result, small as its share is."""
    dim, heads = 64, 4
    p = Pair(cuda, [length], page=32, dim=dim)
    k, v = randn((length, 2, dim), "sink k") * 0.1, randn((length, 2, dim), "sink v")
    k[:, :, 0], k[0], v[0] = 0, 0, 0
    k[0, :, 0] = 8
    p.plain.update(k, v, p.table, [length], [length])
    p.upload()
    q = randn((rows, heads, dim), "sink q", rows)
    q[:, :, 0] = ahead * dim ** 0.5 / 8
    q = q.to(dtype)
    got = p.cache.attention(q.cuda(), p.dtable, ints([length]), dim ** -0.5, row_start=starts([rows]), max_rows=rows, max_len=length).cpu().double()
    want, bound = tight(p.plain, q, p.table[0], length, dim ** -0.5, many=is_many(rows, heads // 2, length))
    assert float((bound / want.abs()).median()) < 0.25, "the bound is to see a result that vanishes"
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,length", [(1, 450), (4, 6000), (200, 450), (70, 3000)])
def test_all_the_weight_on_a_key_of_a_small_block(cuda, dtype, rows, length):
    """The key that takes the weight lies in a page whose values are 2^26 smaller than its neighbours': the result is that key's value."""
    dim, page = 64, 16
    p = Pair(cuda, [length], page=page, dim=dim)
    k, v = randn((length, 2, dim), "small k") * 0.1, randn((length, 2, dim), "small v")
    at = length - rows - 21
    v *= torch.where(torch.arange(length) // page % 3 == at // page % 3, 2.0 ** -16, 2.0 ** 10).reshape(-1, 1, 1)
    k[:, :, 0] = 0
    k[at, :, 0] = 8
    p.plain.update(k, v, p.table, [length], [length])
    p.upload()
    q = randn((rows, 4, dim), "small q", rows)
    q[:, :, 0] = 70.0
    q = q.to(dtype)
    got = p.cache.attention(q.cuda(), p.dtable, ints([length]), dim ** -0.5, row_start=starts([rows]), max_rows=rows, max_len=length).cpu().double()
    want, bound = tight(p.plain, q, p.table[0], length, dim ** -0.5, many=is_many(rows, 2, length))
    big = want.abs() > 2.0 ** -20
    assert float(big.double().mean()) > 0.9 and bool((bound[big] < 0.1 * want[big].abs()).all()), "the bound is to see a result that vanishes"
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,length", [(1, 450), (4, 6000), (16, 4500), (200, 450), (70, 3000)])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e7])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_large_magnitude(cuda, dtype, rows, length, size, sign):
    """Scores up to `size`, all of one sign, the nearest ones apart by more than fp32 rounds: the values of the largest, or the mean of those that share it.

    Queries and keys have one dimension other than 0, so scores are exact but for the roundings that equal ones share; the value scales are equal.  What is left of the
    bound: the sums and the exponential, and the roundings to 11 bits and of the result."""
    dim, heads = 64, 4
    p = Pair(cuda, [length], page=16, dim=dim, tag="large")
    p.plain.k[:] = 0
    p.plain.k[..., 7] = torch.randint(0x70, 0x7F, p.plain.k.shape[:3], dtype=torch.uint8, generator=gen("large", length))  # 128 .. 448, steps of an eighth or less
    p.plain.v[:] = torch.randint(0, 112, p.plain.v.shape, dtype=torch.uint8, generator=gen("large v", length))
    p.plain.scales[..., 0], p.plain.scales[..., 1] = 64.0, 0.5
    p.upload()
    q = torch.zeros((rows, heads, dim))
    q[:, :, 7] = sign * size / (448 * 64 * 0.125)
    q = q.to(dtype)
    got = p.cache.attention(q.cuda(), p.dtable, ints([length]), 0.125, row_start=starts([rows]), max_rows=rows, max_len=length).cpu().double()
    k, v = p.plain.tokens(p.table[0], length)
    for r in range(rows):
        seen = length - rows + r + 1
        for h in range(heads):
            x = k[:seen, h // 2, 7] * float(q[r, h, 7])
            top = x == x.max()
            want, spread = v[:seen, h // 2][top].mean(0), v[:seen, h // 2][top].abs().mean(0)
            bound = (length * 2.0 ** -23 + 2.0 ** -19) * spread + (2.0 ** -11 * spread + 2.0 ** -8 * want.abs() if dtype == BF16 else 0.0)
            assert bool(((got[r, h] - want).abs() <= bound).all()), (r, h)


@pytest.mark.parametrize("rows", [1, 3, 150])
def test_lengths_near_two_to_the_31(cuda, rows):
    """The last tokens of a sequence of 2^31 - 256, seen through a window, are those of a short one; a longer one raises the status."""
    page, dim, window, tail = 64, 64, 400, 12
    p = Pair(cuda, [tail * page], page=page, dim=dim)
    p.fill([tail * page])
    length = 2 ** 31 - 256
    table = torch.zeros((1, 2 ** 31 // page), dtype=torch.int32, device="cuda")
    table[0, length // page - tail:length // page] = p.dtable[0, :tail]
    q = randn((rows, 4, dim), "end", rows)
    args = dict(row_start=starts([rows]), max_rows=rows, window=window)
    for most in (length, 1000):
        got = p.cache.attention(q.cuda(), table, ints([length]), 0.125, max_len=most, **args)
        near(got, q, p, [tail * page], [rows], 0.125, window)
    assert cuda.device_status() == 0
    p.cache.attention(q.cuda(), table, ints([2 ** 31 - 1]), 0.125, max_len=1000, **args)
    with pytest.raises(ops.SharpMindCudaError, match="status 6"):
        cuda.device_status()
