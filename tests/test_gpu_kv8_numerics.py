"""How exact attention over the paged 8-bit cache is where its inputs make that hard: sums that cancel, one key that outweighs all others,
blocks whose scale one key has set, scales far apart.  The bounds do not grow with the number of keys."""
import ctypes as C

import pytest
import torch

from helpers import stream_ptr
from kv8_model import Cache, attention, attention_tolerance
from test_gpu_kv8 import attend_args, ints, status

pytestmark = pytest.mark.gpu


def attend(gpu, liger, cache, lens, q, n, causal=1, max_len=None):
    """`n` new tokens of every sequence, q [len(lens) * n, heads, D]; the result on the CPU, [len(lens) * n, heads, D]."""
    rows, heads, d = q.shape
    cache.to_gpu(liger)
    dq, dl = q.cuda(), ints(lens)
    out = torch.full((rows, heads * d), 7.0, dtype=torch.float16, device="cuda")
    a = attend_args(liger, cache, dq, out, dl, heads, n, len(lens), causal=causal, max_len=max_len)
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    status(gpu)
    return out.cpu().view(rows, heads, d)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_values_that_cancel_show_the_weights(gpu, liger, kind, d, n):
    """Nearly equal weights, and values of alternating sign that all but cancel: the result is small beside sum p |v|, so that what the weights
    were rounded to shows.  The bound is the one of weights in two parts (attention_tolerance), whatever the number of rows."""
    lens = [47, 200, 131, 8]
    cache = Cache(kind, num_pages=30, kv_heads=2, page_size=32, scale_block=16, head_dim=d, slots=4, max_pages=8)
    cache.give_pages(lens)
    for slot, length in enumerate(lens):
        k = torch.randn((length, 2, d), generator=cache.gen)
        sign = torch.where(torch.arange(length) % 2 == 0, 1.0, -1.0)[:, None, None]
        cache.write(0, slot, k, sign * (1.0 + 0.01 * torch.randn((length, 2, d), generator=cache.gen)))
    heads = 4
    q = (torch.randn((len(lens) * n, heads, d), generator=torch.Generator().manual_seed(2)) * 0.03).half()
    got = attend(gpu, liger, cache, lens, q, n)
    for b, length in enumerate(lens):
        want, mixed, size, _ = attention(cache, 0, q[b * n:(b + 1) * n], n, length, b, d ** -0.5, 1)
        off = (got[b * n:(b + 1) * n].double() - want).abs()
        tol = attention_tolerance(want, mixed, size, d)
        assert bool((off <= tol).all()), f"sequence {b}: worst {float((off / tol).max()):.3g} of the tolerance"
