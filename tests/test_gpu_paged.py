"""The paged 8-bit cache on the device: update (codes and scales to the bit), read, and attention against the definition in 64 bits
on the same codes, within the bound that paged_util.attention derives."""
import itertools
import math
import zlib

import pytest
import torch

from sharpmind_b200 import ops, paged
from tests import paged_util

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def gen(*tag):
    return torch.Generator().manual_seed(zlib.crc32(repr(tag).encode()))


def randn(shape, *tag):
    return torch.randn(shape, generator=gen(*tag))


def tables(dim, positions, half=None):
    half = half or dim // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, dtype=torch.float64) / half)
    return angle.cos().float(), angle.sin().float()


class Pair:
    """The device's cache and the plain one, with the same pages."""

    def __init__(self, ctx, lens, kvh=2, dim=128, page=16, extra=3, width=None, tag=0):
        self.page, self.kvh, self.dim = page, kvh, dim
        self.width = width or max(1, max(-(-n // page) for n in lens))
        pages = len(lens) * self.width + extra
        self.table = torch.randperm(pages, generator=gen("table", tag, pages))[:len(lens) * self.width].reshape(len(lens), self.width).to(torch.int32)
        self.plain = paged_util.PlainPages(pages, kvh, page, dim)
        self.cache = paged.PagedKVCache.create(ctx, pages, kvh, dim, page)
        self.upload()
        self.dtable = self.table.cuda()

    def upload(self):
        self.cache.k.view(torch.uint8).copy_(self.plain.k)
        self.cache.v.view(torch.uint8).copy_(self.plain.v)
        self.cache.scales.copy_(self.plain.scales)

    def update(self, lens, rows, k, v, **kw):
        """Both sides; `lens` with the new rows."""
        pos = self.plain.update(k, v, self.table, lens, rows, kw.get("cos"), kw.get("sin"), kw.get("neox", True))
        dkw = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
        out = self.cache.Update(k.cuda(), v.cuda(), self.dtable, ints(lens), row_start=starts(rows), **dkw)
        return pos, out

    def fill(self, lens, tag=0):
        """Tokens of every sequence, written by the plain side."""
        n = sum(lens)
        self.plain.update(randn((n, self.kvh, self.dim), "k", tag, n), randn((n, self.kvh, self.dim), "v", tag, n), self.table, lens, lens)
        self.upload()

    def same(self):
        assert torch.equal(self.cache.scales.cpu().view(torch.int32).masked_fill(self.plain.scales.isnan(), 0), self.plain.scales.view(torch.int32).masked_fill(self.plain.scales.isnan(), 0))
        assert torch.equal(self.cache.scales.cpu().isnan(), self.plain.scales.isnan())
        assert torch.equal(self.cache.k.cpu().view(torch.uint8), self.plain.k)
        assert torch.equal(self.cache.v.cpu().view(torch.uint8), self.plain.v)


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def starts(rows):
    return None if all(n == 1 for n in rows) else ints([0, *itertools.accumulate(rows)])


def near(got, q, pair, lens, rows, scale, window=0):
    want, bound = paged_util.attention(pair.plain, q, pair.table, lens, rows, scale, window, device="cuda")
    got = got.cpu().double()
    n = sum(rows)
    assert torch.equal(got[:n].isnan(), want[:n].isnan())
    off = ((got[:n] - want[:n]).abs() - bound[:n]).nan_to_num(-1.0)
    assert off.max() <= 0 if n else True, (off.max(), (got[:n] - want[:n]).abs().nan_to_num().max())


# ---- update
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,dim,neox,half", [(16, 128, True, 64), (32, 64, False, 32), (64, 128, True, 16), (64, 64, True, 32), (16, 128, False, 12)])
def test_update_has_the_codes_and_scales_of_the_definition(cuda, dtype, page, dim, neox, half):
    """Steps of ragged rows, growing magnitudes among them: a page begun, continued, filled and left; a sequence without new rows."""
    steps = [[1, 5, 0, page], [1, 1, 1, 1], [page - 1, 3, 2 * page + 3, 0], [1, 1, 1, 1], [2, page, 1, 7]]
    lens = [0, 0, 0, 0]
    p = Pair(cuda, [6 * page] * 4, dim=dim, page=page)
    cos, sin = tables(dim, 6 * page, half)
    for i, rows in enumerate(steps):
        lens = [a + b for a, b in zip(lens, rows)]
        n = sum(rows)
        size = torch.exp2(1.7 * randn((n, 2, 1), "size", i))
        k, v = (randn((n, 2, dim), "k", i) * size).to(dtype), (randn((n, 2, dim), "v", i) * size * 3).to(dtype)
        q = randn((n, 6, dim), "q", i).to(dtype)
        pos, out = p.update(lens, rows, k, v, cos=cos, sin=sin, neox=neox, q=q)
        p.same()
        want = torch.stack([paged_util.rotate(q[r].float(), pos[r], cos, sin, neox) for r in range(n)]).to(dtype)
        assert torch.equal(out.cpu(), want)


def test_update_of_blocks_without_magnitude_and_with_the_largest(cuda):
    """Zeros take the smallest scale; 448 2^k fits its own power, the next number does not; values under the smallest code are zeros."""
    p = Pair(cuda, [64], page=16)
    for value in [0.0, 448.0, float(torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))), 448.0 * 2.0 ** -40, 1e-20, 3e38, 1.0, 2.0 ** -60]:
        x = torch.full((1, 2, 128), value)
        x[0, 1] *= -1
        p.update([1], [1], x, x / 2)
        p.same()
    p.update([2], [1], torch.full((1, 2, 128), 1e30), torch.zeros((1, 2, 128)))  # what was there vanishes under the new scale
    p.same()


def test_update_keeps_an_undefined_block_undefined_until_its_page_starts_over(cuda):
    p = Pair(cuda, [32], page=16)
    x = randn((3, 2, 128), "nan")
    bad = x.clone()
    bad[1, 0, 5], bad[2, 1, 7] = math.nan, math.inf
    p.update([3], [3], bad, x)
    p.same()
    assert bool(p.cache.scales[int(p.table[0, 0]), :, 0].isnan().all()) and not bool(p.cache.scales[int(p.table[0, 0]), :, 1].isnan().any())
    p.update([4], [1], x[:1], x[:1])
    p.same()
    p.update([2], [2], x[:2], x[:2])
    p.same()


def test_update_takes_parts_of_a_joined_product_and_rotates_in_place(cuda):
    heads, kvh, dim, n = 4, 2, 64, 21
    p = Pair(cuda, [40, 30], dim=dim, page=32)
    cos, sin = tables(dim, 64)
    joined = randn((n, (heads + 2 * kvh) * dim), "joined").to(BF16).cuda().reshape(n, heads + 2 * kvh, dim)
    q, k, v = joined[:, :heads], joined[:, heads:heads + kvh], joined[:, heads + kvh:]
    rows, lens = [20, 1], [33, 30]
    p.fill([13, 29])
    pos = p.plain.update(k.cpu(), v.cpu(), p.table, lens, rows, cos, sin)
    got = p.cache.Update(k, v, p.dtable, ints(lens), row_start=starts(rows), cos=cos.cuda(), sin=sin.cuda(), q=q)
    want = torch.stack([paged_util.rotate(q[r].cpu().float(), pos[r], cos, sin, True) for r in range(n)]).to(BF16)
    assert torch.equal(got.cpu(), want)
    p.same()
    same = q.contiguous()
    assert p.cache.Update(k, v, p.dtable, ints(lens), row_start=starts(rows), cos=cos.cuda(), sin=sin.cuda(), q=same, q_out=same) is same
    assert torch.equal(same.cpu(), want)


def test_read_gives_the_values(cuda):
    for page, dim, dtype in [(16, 128, F32), (32, 64, BF16), (64, 128, BF16), (64, 64, F32)]:
        p = Pair(cuda, [70, 5, 3 * page], dim=dim, page=page)
        p.fill([70, 5, 3 * page])
        ids = torch.tensor([int(p.table[0, 0]), int(p.table[2, 1]), int(p.table[0, 0])], dtype=torch.int32)
        k, v = p.cache.read(ids.cuda(), dtype)
        for i, pid in enumerate(ids.tolist()):
            wk, wv = p.plain.values(pid)
            assert torch.equal(k[i].cpu(), wk.to(dtype)) and torch.equal(v[i].cpu(), wv.to(dtype))
        k, v = p.cache.read(ids[:0].cuda(), dtype)
        assert k.shape[0] == 0


# ---- attention
SHAPES = [(4, 2, 128, 16), (8, 2, 64, 32), (7, 1, 128, 64), (6, 6, 64, 16), (32, 2, 128, 32), (40, 2, 64, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kvh,dim,page", SHAPES)
def test_attention_of_single_tokens(cuda, dtype, heads, kvh, dim, page):
    """Lengths of nothing, one, around the page and the tiles, and long ones, in one batch; undefined codes behind every length."""
    lens = [0, 1, page - 1, page, page + 1, 63, 64, 65, 127, 129, 700, 1500]
    p = Pair(cuda, lens, kvh=kvh, dim=dim, page=page)
    p.fill(lens)
    q = randn((len(lens), heads, dim), "q", heads, dim).to(dtype)
    for window in (0, 1, 50, 64, 1000):
        got = p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, window=window)
        near(got, q, p, lens, [1] * len(lens), dim ** -0.5, window)
        assert not bool(got[0].any())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kvh,dim,page", SHAPES)
@pytest.mark.parametrize("rows,lens", [([2, 3, 1, 0, 2], [300, 3, 65, 40, 2]), ([5] * 3, [5, 1100, 64]), ([9, 16, 7], [129, 16, 400]), ([33], [500])])
def test_attention_of_a_few_rows(cuda, dtype, heads, kvh, dim, page, rows, lens):
    p = Pair(cuda, lens, kvh=kvh, dim=dim, page=page)
    p.fill(lens)
    q = randn((sum(rows), heads, dim), "q", heads, dim).to(dtype)
    for window in (0, 37):
        got = p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, row_start=starts(rows), max_rows=max(rows), max_len=max(lens), window=window)
        near(got, q, p, lens, rows, dim ** -0.5, window)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kvh,dim,page", SHAPES)
@pytest.mark.parametrize("rows,lens", [([128], [128]), ([300, 1, 0, 77], [300, 900, 12, 333]), ([257, 130], [1000, 131])])
def test_attention_of_prompts(cuda, dtype, heads, kvh, dim, page, rows, lens):
    p = Pair(cuda, lens, kvh=kvh, dim=dim, page=page)
    p.fill(lens)
    q = randn((sum(rows), heads, dim), "q", heads, dim).to(dtype)
    for window in (0, 100):
        got = p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, row_start=starts(rows), window=window)
        near(got, q, p, lens, rows, dim ** -0.5, window)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 4, 200])
def test_attention_where_scores_and_scales_lie_far_apart(cuda, dtype, rows):
    """One key that takes all the weight, pages whose scales differ by 2^30, a page of zeros, large queries: nothing overflows and nothing vanishes."""
    length, dim = 450, 128
    p = Pair(cuda, [length], page=16, dim=dim)
    size = torch.exp2(torch.randint(-18, 12, (-(-length // 16), 1, 1), generator=gen("far")).float()).repeat_interleave(16, 0)[:length]
    k, v = randn((length, 2, dim), "kf") * 0.3, randn((length, 2, dim), "vf") * size
    v[160:176] = 0
    k[77] *= 30
    p.plain.update(k, v, p.table, [length], [length])
    p.upload()
    q = (randn((rows, 4, dim), "qf") * torch.exp2(torch.arange(rows * 4).reshape(rows, 4, 1) % 9 - 4.0)).to(dtype)
    got = p.cache.attention(q.cuda(), p.dtable, ints([length]), dim ** -0.5, row_start=starts([rows]))
    near(got, q, p, [length], [rows], dim ** -0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 3, 150])
def test_undefined_values_reach_the_rows_that_see_them_and_no_others(cuda, dtype, rows):
    """A page whose keys, and one whose values, hold an undefined number; a window that hides them from later rows; causal rows before them."""
    length, page, dim = 400, 16, 64
    p = Pair(cuda, [length, 200], page=page, dim=dim)
    p.fill([length, 200])
    p.plain.scales[int(p.table[0, 20]), 0, 0] = math.nan  # tokens 320 .. 335 of head 0
    p.plain.scales[int(p.table[0, 22]), 1, 1] = math.nan  # tokens 352 .. 367 of head 1
    p.upload()
    q = randn((rows + 1, 4, dim), "qn").to(dtype)
    for window in (0, 40, 60):
        got = p.cache.attention(q.cuda(), p.dtable, ints([length, 200]), dim ** -0.5, row_start=ints([0, rows, rows + 1]), max_rows=rows, window=window)
        near(got, q, p, [length, 200], [rows, 1], dim ** -0.5, window)


def test_rows_behind_the_last_sequence_stay_and_stride_is_read(cuda):
    heads, dim, lens, rows = 4, 64, [90, 200], [30, 5]
    p = Pair(cuda, lens, dim=dim, page=32)
    p.fill(lens)
    wide = randn((50, 3 * heads, dim), "wide").cuda()
    q = wide[:, heads:2 * heads]
    for most in (30, None):
        out = torch.full((50, heads, dim), 7.0, device="cuda")
        p.cache.attention(q, p.dtable, ints(lens), dim ** -0.5, row_start=starts(rows), max_rows=most, out=out)
        assert bool((out[35:] == 7.0).all())
        near(out, q.cpu(), p, lens, rows, dim ** -0.5)
    before = [x.clone() for x in (p.cache.k.view(torch.uint8), p.cache.v.view(torch.uint8))]
    k = randn((50, 2, dim), "behind")
    p.plain.update(k, k, p.table, lens, rows)
    p.cache.Update(k.cuda(), k.cuda(), p.dtable, ints(lens), row_start=starts(rows))
    p.same()
    assert not torch.equal(before[0], p.cache.k.view(torch.uint8))


def test_pages_may_be_shared_by_readers(cuda):
    p = Pair(cuda, [64, 64, 64], page=16)
    p.fill([64, 64, 64])
    p.table[1, :2], p.table[2, :3] = p.table[0, :2], p.table[0, :3]
    p.dtable = p.table.cuda()
    q = randn((3, 4, 128), "shared")
    near(p.cache.attention(q.cuda(), p.dtable, ints([64, 60, 33]), 0.1), q, p, [64, 60, 33], [1, 1, 1], 0.1)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_run_of_them_together(cuda, dtype):
    """Two prompts enter and are attended to, then steps of one token each, then drafts that are taken back and written over: as a server goes."""
    heads, kvh, dim, page = 4, 2, 128, 16
    p = Pair(cuda, [400, 400], page=page, dim=dim)
    cos, sin = tables(dim, 400)
    lens = [0, 0]
    for i, rows in enumerate([[150, 37], [1, 1], [1, 1], [4, 4], [1, 1], [60, 1]]):
        lens = [a + b for a, b in zip(lens, rows)]
        n = sum(rows)
        k, v, q = ((randn((n, h, dim), name, i) * (1 + i)).to(dtype) for name, h in (("k", kvh), ("v", kvh), ("q", heads)))
        _, turned = p.update(lens, rows, k, v, cos=cos, sin=sin, q=q)
        p.same()
        got = p.cache.attention(turned, p.dtable, ints(lens), dim ** -0.5, row_start=starts(rows), max_rows=max(rows), max_len=max(lens))
        near(got, turned.cpu(), p, lens, rows, dim ** -0.5)
        if rows == [4, 4]:
            lens = [n - 2 for n in lens]


@pytest.mark.parametrize("dtype,heads,dim", [(F32, 16, 128), (BF16, 16, 128), (F32, 8, 64), (BF16, 8, 64)])
def test_prompts_back_to_back(cuda, dtype, heads, dim):
    """Two lengths in turn without a pause, every CTA's steps many: each result has its own bits again and again, and no wait is given up."""
    p = Pair(cuda, [1500, 1100], kvh=4, dim=dim, page=64)
    p.fill([1500, 1100])
    q = randn((777, heads, dim), "back", heads).to(dtype).cuda()
    calls = [([777, 0], [777, 1100]), ([500, 277], [1500, 900])]
    first = []
    for i in range(40):
        rows, lens = calls[i % 2]
        got = p.cache.attention(q, p.dtable, ints(lens), dim ** -0.5, row_start=starts(rows), max_rows=max(rows))
        if i < 2:
            near(got, q.cpu(), p, lens, rows, dim ** -0.5)
            first.append(got)
        else:
            assert torch.equal(got, first[i % 2])
    assert cuda.device_status() == 0


@pytest.mark.parametrize("dtype,heads,kvh,dim", [(F32, 8, 8, 64), (BF16, 32, 8, 128), (BF16, 16, 8, 64)])
def test_batches_of_lengths_far_apart(cuda, dtype, heads, kvh, dim):
    """Runs that cut segments and runs that hold many: the same bits each time, with the call's longest length put too short and too long."""
    lens = [20000, 3, 0, 9000, 700, 15000, 64, 5000, 1, 30000]
    p = Pair(cuda, lens, kvh=kvh, dim=dim, page=64, tag="asked")
    p.plain.k[:] = torch.randint(0, 112, p.plain.k.shape, dtype=torch.uint8, generator=gen("codes")) | (torch.randint(0, 2, p.plain.k.shape, dtype=torch.uint8, generator=gen("signs")) << 7)
    p.plain.v[:] = p.plain.k.transpose(2, 3).flip(2)
    p.plain.scales[:] = torch.exp2(torch.randint(-9, -5, p.plain.scales.shape, generator=gen("scales")).float())
    p.upload()
    q = randn((len(lens), heads, dim), "asked", heads).to(dtype)
    first = p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5)
    near(first, q, p, lens, [1] * len(lens), dim ** -0.5)
    for _ in range(20):
        assert torch.equal(first, p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5))
    # shorter and longer than the call says
    for long in (4000, 500000):
        near(p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, max_len=long), q, p, lens, [1] * len(lens), dim ** -0.5)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("dtype,rows,window", [(F32, 1, 0), (BF16, 1, 300), (BF16, 4, 0), (F32, 3, 130)])
def test_many_segments_of_some_length(cuda, dtype, rows, window):
    """More segments than blocks of threads on the device, up to 32 tiles each: several whole ones to a block; among them empty sequences and single keys."""
    lens = [[2048, 0, 1, 700, 1999, 65, 64, 1300][i % 8] for i in range(168)]
    count = [min(rows, n) for n in lens]
    p = Pair(cuda, lens, kvh=2, dim=64, page=32, tag="many")
    p.fill(lens)
    q = randn((sum(count), 4, 64), "many", rows).to(dtype)
    start = [0]
    for n in count:
        start.append(start[-1] + n)
    got = p.cache.attention(q.cuda(), p.dtable, ints(lens), 0.125, row_start=ints(start), max_rows=rows, window=window)
    near(got, q, p, lens, count, 0.125, window)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kvh,most,batch,window", [(2, 5, 6, 0), (1, 16, 7, 0), (2, 9, 5, 700), (2, 5, 72, 0), (1, 12, 160, 0)])
def test_drafts_over_long_caches(cuda, dtype, dim, kvh, most, batch, window):
    """17 to 64 (row, head) pairs of a sequence, beside sequences with fewer and with none; long enough for the form that takes them in sixteens."""
    lens = [[4500, 70, 1025, 0, 2000, 3, 4096][i % 7] for i in range(batch)]
    count = [min([most, 1, most - 1, 3, 0, 2][i % 6], n) for i, n in enumerate(lens)]
    p = Pair(cuda, lens, kvh=kvh, dim=dim, page=32, tag="drafts")
    p.fill(lens)
    group = 4
    q = randn((sum(count), kvh * group, dim), "drafts", most).to(dtype)
    args = dict(row_start=starts(count), max_rows=most, window=window)
    got = p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, **args)
    near(got, q, p, lens, count, dim ** -0.5, window)
    assert torch.equal(got, p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, **args))
    # a longest length that says less than there is, and so the forms for shorter ones; one that says all that there may be
    for long in (600, 2048, 2 ** 31 - 1):
        near(p.cache.attention(q.cuda(), p.dtable, ints(lens), dim ** -0.5, max_len=long, **args), q, p, lens, count, dim ** -0.5, window)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_other_scales(cuda, dtype, rows, scale):
    """Nothing but the mean, the order turned round, and a sharp softmax; among queries a row of zeros, tiny ones and large ones."""
    lens = [333, 64]
    p = Pair(cuda, lens, dim=64, page=16)
    p.fill(lens)
    q = randn((2 * rows, 6, 64), "scales", rows)
    q[0] = 0
    q[1] *= 1e-30
    q[-1, 3] *= 1e4
    q = q.to(dtype)
    got = p.cache.attention(q.cuda(), p.dtable, ints(lens), scale, row_start=starts([rows, rows]), max_rows=rows)
    want, bound = paged_util.attention(p.plain, q, p.table, lens, [rows, rows], scale, device="cuda")
    if scale < 0:  # (the bound's sizes are of the scale's magnitude)
        bound = paged_util.attention(p.plain, -q, p.table, lens, [rows, rows], -scale, device="cuda")[1]
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("rows", [1, 50])
def test_a_cache_of_more_than_four_gigabytes(cuda, rows):
    """Pages whose codes lie behind 2^32 bytes, beside pages in front of them."""
    kvh, page, dim, pages, heads, length = 8, 64, 128, 68000, 16, 200
    cache = paged.PagedKVCache.create(cuda, pages, kvh, dim, page)
    assert cache.k.numel() > 1 << 32
    plain = paged_util.PlainPages(4, kvh, page, dim)
    far = ints([[pages - 1, 3, pages - 2, 65536]])
    k, v = randn((length, kvh, dim), "far k"), randn((length, kvh, dim), "far v")
    plain.update(k, v, [[0, 1, 2, 3]], [length], [length])
    cache.Update(k.cuda(), v.cuda(), far, ints([length]), row_start=ints([0, length]))
    gk, gv = cache.read(far[0])
    for i in range(3):
        assert torch.equal(gk[i].cpu(), plain.values(i)[0]) and torch.equal(gv[i].cpu(), plain.values(i)[1])
    q = randn((rows, heads, dim), "far q")
    got = cache.attention(q.cuda(), far, ints([length]), 0.1, row_start=None if rows == 1 else ints([0, rows]))
    want, bound = paged_util.attention(plain, q, [[0, 1, 2, 3]], [length], [rows], 0.1)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


# ---- where and when it runs
@pytest.mark.parametrize("rows", [1, 3, 140])
def test_captured_calls_serve_what_the_arrays_hold(cuda, rows):
    """One graph of an update and its attention, replayed as the sequences grow, while a second graph over other pages replays on another stream."""
    heads, dim, lens0 = 4, 64, [10, 200]
    pairs, graphs, bufs = [], [], []
    for g in range(2):
        p = Pair(cuda, [900, 900], dim=dim, page=32, tag=g)
        p.fill([n + 7 * g for n in lens0], tag=g)
        lens = ints([n + 7 * g + rows for n in lens0])
        k, v, q = (randn((2 * rows, h, dim), name, g).cuda() for name, h in (("k", 2), ("v", 2), ("q", heads)))
        start = starts([rows, rows])
        out = torch.zeros_like(q)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                p.cache.Update(k, v, p.dtable, lens, row_start=start)
                p.cache.attention(q, p.dtable, lens, 0.125, row_start=start, max_rows=rows, max_len=900, out=out)
        pairs.append(p), graphs.append((graph, stream)), bufs.append((lens, k, v, q, out, start))  # (a graph keeps none of its arguments alive)
    torch.cuda.synchronize()
    host = [[n + 7 * g + rows for n in lens0] for g in range(2)]
    for step in range(4):
        for g in range(2):
            k = randn((2 * rows, 2, dim), "step", step, g)
            bufs[g][0].copy_(torch.tensor(host[g], dtype=torch.int32)), bufs[g][1].copy_(k), bufs[g][2].copy_(k * 2)
        torch.cuda.synchronize()
        for graph, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for g in range(2):
            k = randn((2 * rows, 2, dim), "step", step, g)
            pairs[g].plain.update(k, k * 2, pairs[g].table, host[g], [rows, rows])
            pairs[g].same()
            near(bufs[g][4], bufs[g][3].cpu(), pairs[g], host[g], [rows, rows], 0.125)
            host[g] = [n + rows for n in host[g]]


@pytest.mark.parametrize("rows", [1, 150])
def test_the_same_call_has_the_same_bits(cuda, rows):
    lens = [3000, 10, 777]
    p = Pair(cuda, lens, page=64)
    p.fill(lens)
    q = randn((3 * rows, 8, 128), "bits").cuda()
    lens = [max(n, rows) for n in lens]
    if rows > 1:
        lens = [3000, 150, 777]
        p.fill(lens)
    first = p.cache.attention(q, p.dtable, ints(lens), 0.1, row_start=starts([rows] * 3), max_rows=rows)
    for _ in range(5):
        assert torch.equal(first, p.cache.attention(q, p.dtable, ints(lens), 0.1, row_start=starts([rows] * 3), max_rows=rows))


def test_on_another_stream(cuda):
    lens = [500, 90]
    p = Pair(cuda, lens, page=32)
    p.fill(lens)
    q = randn((2, 4, 128), "stream")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = p.cache.attention(q.cuda(non_blocking=False), p.dtable, ints(lens), 0.1)
    side.synchronize()
    near(got, q, p, lens, [1, 1], 0.1)


def test_two_threads_on_their_own_streams(cuda):
    """Calls at the same time, each with its own pages and work space."""
    import threading

    pairs, wants, faults = [], [], []
    for i in range(2):
        p = Pair(cuda, [1200, 300], kvh=4, dim=64, page=32, tag=("thread", i))
        p.fill([1200, 300], tag=("thread", i))
        pairs.append((p, randn((2, 16, 64), "t1", i).cuda(), randn((140, 16, 64), "t2", i).cuda(), ints([1200, 300]), ints([0, 100, 140])))
        wants.append((p.cache.attention(pairs[i][1], p.dtable, pairs[i][3], 0.125), p.cache.attention(pairs[i][2], p.dtable, pairs[i][3], 0.125, row_start=pairs[i][4])))
    torch.cuda.synchronize()

    def work(i):
        p, one, many, lens, start = pairs[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                a, b = p.cache.attention(one, p.dtable, lens, 0.125), p.cache.attention(many, p.dtable, lens, 0.125, row_start=start)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(a, wants[i][0]) and torch.equal(b, wants[i][1])):
                    faults.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults


# ---- what it refuses
def test_pages_lengths_and_rows_out_of_range_raise_the_status(cuda):
    """Nothing outside of the arrays is touched, the other sequences are served, and the status tells."""
    p = Pair(cuda, [200, 200, 200], page=16, extra=1)
    p.fill([200, 200, 200])
    q = randn((3, 4, 128), "bad")
    k = randn((3, 2, 128), "badk")
    spoiled = [(torch.tensor([-1]), [200, 200, 200]), (torch.tensor([1 << 30]), [200, 200, 200]), (None, [200, 5000, 200]), (None, [200, -3, 200])]
    for page, lens in spoiled:
        table = p.table.clone()
        if page is not None:
            table[1, 12] = page[0]
        got = p.cache.attention(q.cuda(), table.cuda(), ints(lens), 0.1)
        with pytest.raises(ops.SharpMindCudaError, match="status 6"):
            cuda.device_status()
        near(got[::2], q[::2], _Rows(p, [0, 2]), [200, 200], [1, 1], 0.1)
        before = p.cache.k.view(torch.uint8).clone()
        p.cache.Update(k.cuda(), k.cuda(), table.cuda(), ints(lens))
        with pytest.raises(ops.SharpMindCudaError, match="status 6"):
            cuda.device_status()
        changed = (before != p.cache.k.view(torch.uint8)).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= {int(p.table[0, 12]), int(p.table[2, 12])}
        p.upload()
    big = randn((150, 4, 128), "badrows").cuda()
    for start in ([0, 150, 400, 450], [-5, 20, 30, 150], [0, 60, 40, 150]):
        p.cache.attention(big, p.dtable, ints([200, 200, 200]), 0.1, row_start=ints(start))
        p.cache.Update(big[:, :2], big[:, :2], p.dtable, ints([200, 200, 200]), row_start=ints(start))
        with pytest.raises(ops.SharpMindCudaError, match="status 6"):
            cuda.device_status()
    # more rows than the call says, and positions behind the rotation's tables
    p.upload()
    p.cache.attention(big[:40], p.dtable, ints([200, 200, 200]), 0.1, row_start=ints([0, 20, 39, 40]), max_rows=2)
    with pytest.raises(ops.SharpMindCudaError, match="status 6"):
        cuda.device_status()
    cos, sin = tables(128, 150)
    p.cache.Update(k.cuda(), k.cuda(), p.dtable, ints([200, 140, 100]), cos=cos.cuda(), sin=sin.cuda(), q=q.cuda())
    with pytest.raises(ops.SharpMindCudaError, match="status 6"):
        cuda.device_status()
    k1, v1 = p.cache.read(ints([0, -1, p.cache.pages]))
    with pytest.raises(ops.SharpMindCudaError, match="status 6"):
        cuda.device_status()
    assert not bool(k1[1:].any()) and not bool(v1[1:].any())


class _Rows:
    """Some of a pair's sequences."""

    def __init__(self, pair, which):
        self.plain, self.table = pair.plain, pair.table[which]


def test_calls_with_nothing_to_do(cuda):
    p = Pair(cuda, [20], page=16)
    p.fill([20])
    none = torch.empty((0, 4, 128), device="cuda")
    table, lens = torch.empty((0, 4), dtype=torch.int32, device="cuda"), ints([])
    assert p.cache.attention(none, table, lens, 0.1).shape == (0, 4, 128)
    p.cache.Update(none[:, :2], none[:, :2], table, lens)
    assert p.cache.attention(none, p.dtable, ints([20]), 0.1, row_start=ints([0, 0])).shape == (0, 4, 128)
    p.same()


def test_the_library_refuses_what_it_has_no_kernel_for(cuda):
    """The C entry points themselves, whose checks come before any launch."""
    import ctypes as C

    p = Pair(cuda, [20], page=16)
    lib, s = cuda.lib, paged._Seqs(p.dtable.data_ptr(), ints([20]).data_ptr(), None, 1, p.width, 1)
    x = torch.zeros((1, 4, 128), device="cuda")

    def attend(kv=p.cache._kv, seqs=s, dtype=0, q=x.data_ptr(), stride=512, out=x.data_ptr(), heads=4, window=0, most=1, long=20):
        n = lib.smc_paged_attention_work(cuda.h, C.byref(kv), 1, 1, heads, most, long)
        work = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        return lib.smc_paged_attention_dev(cuda.h, C.byref(kv), C.byref(seqs), dtype, q, stride, out, heads, 0.1, window, most, long, work.data_ptr(), max(n, 0), None)

    def changed(**kw):
        kv = paged._Kv.from_buffer_copy(p.cache._kv)
        for name, value in kw.items():
            setattr(kv, name, value)
        return kv

    assert attend() == 0
    assert attend(dtype=1) == 2 and attend(kv=changed(page=48)) == 2 and attend(kv=changed(head_dim=96)) == 2
    assert attend(kv=changed(k=None)) == 1 and attend(kv=changed(v=p.cache.v.data_ptr() + 4)) == 1 and attend(kv=changed(pages=0)) == 1
    assert attend(heads=3) == 1 and attend(window=-1) == 1 and attend(most=-1) == 1 and attend(long=-1) == 1
    assert attend(q=x.data_ptr() + 4) == 1 and attend(stride=256) == 1 and attend(stride=514) == 1 and attend(out=None) == 1
    assert attend(seqs=paged._Seqs(p.dtable.data_ptr(), None, None, 1, p.width, 1)) == 1
    assert attend(seqs=paged._Seqs(p.dtable.data_ptr(), p.dtable.data_ptr(), None, 1, p.width, 2)) == 1
    torch.cuda.synchronize()
