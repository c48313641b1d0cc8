"""liger_kv8_append: entries and pages that must not be written, beside others that must."""
import ctypes as C

import pytest
import torch

from helpers import stream_ptr
from kv8_model import Cache, append
from test_gpu_kv8 import BAD_INDEX, ints, same_cache, status

pytestmark = pytest.mark.gpu


def call(gpu, liger, cache, k, v, first, slots, offsets, q_len, total):
    a = liger.Kv8AppendArgs()
    hold = k.cuda(), v.cuda(), ints(first), ints(slots), ints(offsets)
    a.k, a.v, a.positions, a.slots, a.q_offsets = (t.data_ptr() for t in hold)
    a.batch, a.q_len, a.total_tokens = len(first), q_len, total
    a.token_stride, a.head_stride = cache.kv_heads * cache.head_dim, cache.head_dim
    liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
    torch.cuda.synchronize()


def small_cache(liger, kind="int8"):
    cache = Cache(kind, num_pages=16, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=3, max_pages=4)
    cache.give_pages([128, 128, 128])
    cache.fill([10, 20, 30])
    return cache.to_gpu(liger)


@pytest.mark.parametrize("offsets,first,q_len", [
    ([0, 9, 12], [10, 10], 5),           # the first entry brings more than q_len tokens
    ([9, 20, 12], [10, 10], 12),         # its rows end behind the call's last one, and the second's begin behind their end: both left out
    ([0, 3, 6], [126, 10], 5),           # its tokens end behind the table's row
    ([0, 3, 6], [-1, 10], 5),
    ([0, 3, 6], [2 ** 31 - 2, 10], 5)])
def test_an_entry_that_is_left_out_does_not_claim_its_slot(gpu, liger, offsets, first, q_len):
    cache = small_cache(liger)
    total = 14
    k, v = (torch.randn((total, 2, 64), generator=torch.Generator().manual_seed(i)).half() for i in range(2))
    call(gpu, liger, cache, k, v, first, [1, 1], offsets, q_len, total)
    status(gpu, BAD_INDEX)
    lo, hi = offsets[1:]
    if lo <= hi:
        append(cache, 0, 1, first[1], k[lo:hi], v[lo:hi])
    same_cache(cache)


def test_of_two_entries_that_count_the_first_is_written(gpu, liger):
    """An entry that is left out, one without tokens, one that counts, and one behind it, all of one slot."""
    cache = small_cache(liger, "e4m3")
    k, v = (torch.randn((12, 2, 64), generator=torch.Generator().manual_seed(i)).half() for i in range(2))
    call(gpu, liger, cache, k, v, [200, 0, 20, 20], [1, 1, 1, 1], [0, 3, 3, 8, 12], 5, 12)
    status(gpu, BAD_INDEX)
    append(cache, 0, 1, 20, k[3:8], v[3:8])
    same_cache(cache)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_page_that_two_slots_share_is_not_written(gpu, liger, kind):
    """A branch that goes back into the part that it shares: those tokens are left out, in the pages that are its own they are written, and the other
    branch reads what it did.  Once it has the pages for itself the same call is carried out."""
    cache = Cache(kind, num_pages=16, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=3, max_pages=4)
    cache.give_pages([100])
    cache.fill([100])
    cache.to_gpu(liger)
    space = torch.empty(gpu.liger_kv8_pages_scratch_bytes(cache.by, 1), dtype=torch.uint8, device="cuda")
    args = ints([0]), ints([1]), ints([70])
    liger.check(gpu.liger_kv8_fork(cache.by, *(C.c_void_p(t.data_ptr()) for t in args), 1, None, C.c_void_p(space.data_ptr()), space.numel(), stream_ptr()))
    status(gpu)
    for n in cache.NAMES:
        getattr(cache, n).copy_(cache.dev[n].cpu())
    shared = [int(p) for p in cache.table[1, :2]]
    assert [int(cache.refs[p]) for p in shared] == [2, 2] and int(cache.table[0, 0]) == shared[0]
    k, v = (torch.randn((40, 2, 64), generator=torch.Generator().manual_seed(i)).half() for i in range(2))
    # positions 40 .. 79: 40 .. 63 lie in the second shared page, 64 .. 79 in the slot's own
    call(gpu, liger, cache, k, v, [40], [1], [0, 40], 40, 40)
    status(gpu, BAD_INDEX)
    before = {n: getattr(cache, n)[0, shared[1]].clone() for n in ("k", "v", "ks", "vs")}
    append(cache, 0, 1, 40, k, v)
    for n, t in before.items():
        getattr(cache, n)[0, shared[1]] = t
    same_cache(cache)
    gone = ints([0])
    liger.check(gpu.liger_kv8_free(cache.by, C.c_void_p(gone.data_ptr()), 1, stream_ptr()))
    call(gpu, liger, cache, k, v, [40], [1], [0, 40], 40, 40)
    status(gpu)
    append(cache, 0, 1, 40, k, v)
    same_cache(cache)
