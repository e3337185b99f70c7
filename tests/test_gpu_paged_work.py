"""The work space that a paged attention call asks for: refused where it is not there, kept to where it is."""
import ctypes as C

import pytest
import torch

from sharpmind_b200 import paged
from tests.test_gpu_paged import Pair, ints, near, randn

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def test_calls_of_some_pairs_take_the_form_that_was_measured_faster(cuda):
    """The work space tells the forms apart: runs of sixteen pairs ask for less than pieces of 256.  3 x 16 pairs over 3000 keys and 4 x 16 over 4000 go by sixteens,
    over 2000 and 3000 they do not."""
    kv = paged._Kv(256, 256, 256, 1, 8, 64, 128)

    def need(rows, length):
        return cuda.lib.smc_paged_attention_work(cuda.h, C.byref(kv), 8, 8 * rows, 32, rows, length)

    runs = need(16, 8000)
    for rows, length, sixteens in [(12, 3000, True), (16, 4000, True), (5, 2000, True), (12, 2000, False), (16, 3000, False)]:
        assert (need(rows, length) <= runs) == sixteens, (rows, length)


# heads, rows of a sequence, sequences, tokens: runs with a join, segments of sixteen pairs, pieces of a prompt, and calls that need none
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,each,batch,length,needs", [(8, 1, 2, 5000, True), (8, 2, 3, 3000, True), (8, 16, 2, 4500, True), (8, 40, 2, 2000, True), (8, 1, 2, 400, False),
                                                           (32, 700, 6, 1200, False)])
def test_work_space_is_asked_for_and_kept_to(cuda, dtype, heads, each, batch, length, needs):
    """Null, misaligned and short work space is refused; exactly as much as is asked for, inside of a larger buffer, leaves the bytes around it."""
    kvh, dim, page = 2, 64, 64
    p = Pair(cuda, [length] * batch, kvh=kvh, dim=dim, page=page)
    p.fill([length] * batch)
    rows = each * batch
    q = randn((rows, heads, dim), "work", each).to(dtype)
    dq, out, lens = q.cuda(), torch.empty((rows, heads, dim), dtype=dtype, device="cuda"), ints([length] * batch)
    start = ints(list(range(0, rows + 1, each)))
    seqs = paged._Seqs(p.dtable.data_ptr(), lens.data_ptr(), start.data_ptr(), batch, p.width, rows)
    need = cuda.lib.smc_paged_attention_work(cuda.h, C.byref(p.cache._kv), batch, rows, heads, each, length)
    assert (need > 0) == needs
    guard = 4096
    buffer = torch.full((need + 2 * guard,), 0x5A, dtype=torch.uint8, device="cuda")

    def call(work, size):
        return cuda.lib.smc_paged_attention_dev(cuda.h, C.byref(p.cache._kv), C.byref(seqs), 0 if dtype == F32 else 30, dq.data_ptr(), heads * dim, out.data_ptr(), heads, dim ** -0.5, 0,
                                                each, length, work, size, torch.cuda.current_stream().cuda_stream)

    if needs:
        assert call(None, need) == 1 and call(buffer.data_ptr() + guard, need - 1) == 1 and call(buffer.data_ptr() + guard + 4, need) == 1
        assert bool((buffer == 0x5A).all())
    assert call(buffer.data_ptr() + guard if needs else None, need) == 0
    assert bool((buffer[:guard] == 0x5A).all()) and bool((buffer[guard + need:] == 0x5A).all())
    near(out, q, p, [length] * batch, [each] * batch, dim ** -0.5)
    assert cuda.device_status() == 0
