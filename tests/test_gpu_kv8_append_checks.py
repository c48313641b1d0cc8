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
