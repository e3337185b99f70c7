"""Empty slots of a batch in the paged cache's update and attention."""
import pytest
import torch

from sharpmind_b200 import ops
from tests import paged_util
from tests.test_gpu_paged import Pair, ints, near, randn, tables

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rope", [None, "halves", "neighbours"])
@pytest.mark.parametrize("implied,each", [(True, 1), (False, 1), (False, 3)])
def test_a_padded_batch_is_updated_and_attended_to(cuda, dtype, rope, implied, each):
    """Slots of length 0 among the others, as a batch of a fixed size has them: nothing is written for them, their queries come through as they are, attention
    gives zeros, and no status is raised."""
    heads, kvh, dim, page = 4, 2, 64, 16
    before = [0, 15, 0, 40, 16, 0]
    used = [0, 1, 0, 1, 1, 0]
    lens = [n + each if u else 0 for n, u in zip(before, used)]
    p = Pair(cuda, [64] * 6, kvh=kvh, dim=dim, page=page)
    p.fill(before)
    n = 6 * each
    k, v, q = ((randn((n, h, dim), name, each) * 4).to(dtype) for name, h in (("k", kvh), ("v", kvh), ("q", heads)))
    cos, sin = tables(dim, 64) if rope else (None, None)
    start = None if implied else ints(list(range(0, n + 1, each)))
    there = [r for s in range(6) if used[s] for r in range(s * each, (s + 1) * each)]
    places = p.plain.update(k[there], v[there], p.table, lens, [each * u for u in used], cos, sin, rope != "neighbours")
    kw = {} if rope is None else dict(cos=cos.cuda(), sin=sin.cuda(), neox=rope == "halves")
    turned = p.cache.Update(k.cuda(), v.cuda(), p.dtable, ints(lens), row_start=start, q=q.cuda(), q_out=torch.full_like(q, 7).cuda(), **kw)
    assert cuda.device_status() == 0
    p.same()
    want = q.clone()
    if rope:
        for r, pos in zip(there, places):
            want[r] = paged_util.rotate(q[r].float(), pos, cos, sin, rope == "halves").to(dtype)
    assert torch.equal(turned.cpu(), want)
    got = p.cache.attention(turned, p.dtable, ints(lens), dim ** -0.5, row_start=start, max_rows=each)
    assert cuda.device_status() == 0
    empty = [r for r in range(n) if r not in there]
    assert not bool(got[empty].any())
    near(got[there], turned[there].cpu(), p, lens, [each * u for u in used], dim ** -0.5)


def test_a_batch_of_empty_slots_only_replayed_as_it_fills(cuda):
    """A captured step whose slots are empty at its capture and filled one after the other."""
    p = Pair(cuda, [64] * 3, dim=64, page=16)
    k, v, q = (randn((3, h, 64), name).cuda() for name, h in (("k", 2), ("v", 2), ("q", 4)))
    lens, out = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((3, 4, 64), 7.0, device="cuda")
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        p.cache.Update(k, v, p.dtable, lens)
        p.cache.attention(q, p.dtable, lens, 0.125, max_len=64, out=out)
    host = [0, 0, 0]
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert cuda.device_status() == 0
        live = [s for s in range(3) if host[s]]
        if live:
            p.plain.update(k[live].cpu(), v[live].cpu(), p.table, host, [int(n > 0) for n in host])
        p.same()
        near(out[live], q[live].cpu(), p, host, [int(n > 0) for n in host], 0.125)
        assert not bool(out[[s for s in range(3) if not host[s]]].any())
        host = [n + 1 if n or s <= step else 0 for s, n in enumerate(host)]
        lens.copy_(torch.tensor(host, dtype=torch.int32))


def test_what_is_not_an_empty_slot_still_raises_the_status(cuda):
    """A negative length, and more rows than tokens."""
    p = Pair(cuda, [40, 40], dim=64, page=16)
    p.fill([20, 20])
    k = randn((8, 2, 64), "k").cuda()
    for lens, start in (([20, -1], None), ([20, 2], ints([0, 4, 8]))):
        rows = 2 if start is None else 8
        p.cache.Update(k[:rows], k[:rows], p.dtable, ints(lens), row_start=start)
        with pytest.raises(ops.SharpMindCudaError, match="status 6"):
            cuda.device_status()
