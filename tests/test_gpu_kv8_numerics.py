"""How exact attention over the paged 8-bit cache is where its inputs make that hard: sums that cancel, one key that outweighs all others,
blocks whose scale one key has set, scales far apart.  The bounds do not grow with the number of keys."""
import ctypes as C
import random

import pytest
import torch

from helpers import stream_ptr
from kv8_model import Cache, attention, attention_tolerance
from test_gpu_kv8 import attend_args, ints, status

pytestmark = pytest.mark.gpu
TIMEOUT = 1


def attend(gpu, liger, cache, lens, q, n, causal=1, max_len=None, offsets=None):
    """`n` new tokens of every sequence, or as the offsets say and `n` at most, q [tokens, heads, D]; the result on the CPU, [tokens, heads, D]."""
    rows, heads, d = q.shape
    cache.to_gpu(liger)
    dq, dl, do = q.cuda(), ints(lens), ints(offsets) if offsets else None
    out = torch.full((rows, heads * d), 7.0, dtype=torch.float16, device="cuda")
    a = attend_args(liger, cache, dq, out, dl, heads, n, len(lens), offsets=do, total=rows, causal=causal, max_len=max_len)
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


@pytest.fixture
def short_waits(gpu, liger):
    liger.check(gpu.liger_set_wait_budget_ms(1))
    yield
    liger.check(gpu.liger_set_wait_budget_ms(2000))


def long_sequence_of_few_pages(liger, times, q_len, group, kv_heads=10):
    """A sequence whose table names the same 1024 tokens `times` times over: attention without a causal mask gives what those tokens alone
    give.  Also queries for it."""
    cache = Cache("int8", num_pages=4, kv_heads=kv_heads, page_size=256, scale_block=128, head_dim=64, slots=1, max_pages=4 * times)
    cache.give_pages([1024])
    cache.fill([1024])
    cache.table[0] = cache.table[0, :4].repeat(times)
    cache.to_gpu(liger)
    q = torch.randn((q_len, kv_heads * group, 64), generator=torch.Generator().manual_seed(4)).half()
    return cache, q


def test_waits_that_run_out_write_nothing_beside_the_result(gpu, liger, short_waits):
    """Shares of several milliseconds with a budget of one for each wait, and a workspace that holds numbers which look like records of an
    earlier call.  Either the call is answered, or it says that a wait ran out; memory around its rows stays as it was."""
    cache, q = long_sequence_of_few_pages(liger, 200, q_len=160, group=16)
    heads, width = 160, 160 * 64
    space = torch.full((160 + 2 * 64, width), 7.0, dtype=torch.float16, device="cuda")
    out = space[64:-64]
    dq, dl = q.cuda(), ints([1024 * 200])
    a = attend_args(liger, cache, dq, out, dl, heads, 160, 1, causal=0)
    for old in (0x01010101, 3, 0x00012345):
        a.keep.view(torch.int32).fill_(old)
        liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
        torch.cuda.synchronize()
        st = (C.c_uint * 4)()
        code = gpu.liger_device_status(C.byref(st))
        gpu.liger_device_status_clear()
        assert code in (0, TIMEOUT), list(st)
        assert bool((space[:64] == 7.0).all()) and bool((space[-64:] == 7.0).all())
        if code == 0:
            want, mixed, size, _ = attention(cache, 0, q, 160, 1024, 0, 64 ** -0.5, 0)
            off = (out.cpu().double().view(160, heads, 64) - want).abs()
            assert bool((off <= attention_tolerance(want, mixed, size, 64)).all())


@pytest.mark.parametrize("times", [200, 1000])
def test_a_short_budget_suffices_for_waits_over_long_tiles(gpu, liger, short_waits, times):
    """The budget is for a wait in which nothing goes on: a tile of a million keys takes longer than a millisecond and is answered."""
    cache, q = long_sequence_of_few_pages(liger, times, q_len=160 if times == 200 else 20, group=16)
    n, heads = q.shape[:2]
    want, mixed, size, _ = attention(cache, 0, q, n, 1024, 0, 64 ** -0.5, 0)
    got = attend(gpu, liger, cache, [1024 * times], q, n, causal=0)
    off = (got.double() - want).abs()
    assert bool((off <= attention_tolerance(want, mixed, size, 64)).all())


@pytest.mark.parametrize("group", [1, 60])
def test_more_than_2_to_the_24_keys(gpu, liger, group):
    cache, q = long_sequence_of_few_pages(liger, 17000, q_len=1, group=group, kv_heads=1)
    want, mixed, size, _ = attention(cache, 0, q, 1, 1024, 0, 64 ** -0.5, 0)
    got = attend(gpu, liger, cache, [1024 * 17000], q, 1, causal=0)
    off = (got.double() - want).abs()
    assert bool((off <= attention_tolerance(want, mixed, size, 64)).all())


# What weights may be off by beside 2^-18 of each (attention_tolerance): two fp16 parts end at 2^-24, off by 2^-25, in units in which a weight at the
# reference score is 2^11 (2^10 with up to 48 rows a key head) and the reference score is no higher than the largest score of the block, of 128 keys (16),
# where that is the largest so far.
def lost_in_a_block(p_top, v_top, keys=128):
    return keys * p_top * v_top * 2.0 ** -25 * 2.0 ** -11


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("below", [17, 21, 25])
@pytest.mark.parametrize("n", [1, 7, 12, 20, 60])
def test_one_key_of_no_value_in_front_of_a_long_tail(gpu, liger, kind, d, below, n):
    """The first key outweighs each of the others by 2^below, and its value is 0: what the result consists of is the tail.  Only the keys that share the
    first one's block may lose bits to it."""
    length = 4000
    cache = Cache(kind, num_pages=64, kv_heads=1, page_size=64, scale_block=16, head_dim=d, slots=1, max_pages=64)
    cache.give_pages([length])
    k, v = torch.randn((length, 1, d), generator=cache.gen) * 0.2, 64.0 + 6.0 * torch.randn((length, 1, d), generator=cache.gen)
    k[:, :, 0] = 0.0
    q = torch.randn((n, 1, d), generator=torch.Generator().manual_seed(6)) * 0.2
    q[:, :, 0] = 4.0
    k[0, 0, 0] = below * d ** 0.5 / (4.0 * 1.4427)
    v[0] = 0.0
    cache.write(0, 0, k, v)
    q = q.half()
    got = attend(gpu, liger, cache, [length], q, n, causal=0).double()
    want, mixed, size, top = attention(cache, 0, q, n, length, 0, d ** -0.5, 0)
    assert 2.0 ** -9 < float(want.min()) and float(want.max()) < 8
    tol = attention_tolerance(want, mixed, size, d) + lost_in_a_block(1.0, top)
    off = (got - want).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the tolerance, {float((off / want).max()):.3g} of the result"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("n,max_len", [(1, 20000), (2, 900), (7, 20000), (20, 20000)])
@pytest.mark.parametrize("falling", [True, False])
def test_value_scales_that_fall_or_rise_with_every_step(gpu, liger, kind, n, max_len, falling):
    """The same with few rows, whose steps are of 16 keys: three sizes in turn."""
    scales = [0.5, 0.5 * 2.0 ** -59.9, 0.5 * 2.0 ** -119.8]
    length = 16 * 50
    cache = Cache(kind, num_pages=50, kv_heads=2, page_size=16, scale_block=16, head_dim=64, slots=1, max_pages=1250)
    cache.give_pages([length])
    cache.fill([length])
    cache.v.random_(60, 120, generator=cache.gen)
    for j in range(50):
        cache.vs[0, int(cache.table[0, j])] = scales[(j if falling else 49 - j) % 3]
    q = (torch.randn((n, 2, 64), generator=torch.Generator().manual_seed(6))).half()
    got = attend(gpu, liger, cache, [length], q, n, causal=0, max_len=max_len).double()
    want, mixed, size, top = attention(cache, 0, q, n, length, 0, 64 ** -0.5, 0)
    tol = attention_tolerance(want, mixed, size, 64) + lost_in_a_block(1.0, top)
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("n", [60])
@pytest.mark.parametrize("falling", [True, False])
def test_value_scales_that_fall_or_rise_step_by_step(gpu, liger, n, falling):
    """Values of one sign, the later blocks' 2^-59.9 and 2^-119.8 of the first ones', or the other way round: the result is the largest blocks' share, a
    number.  One tile is one share here, so that all of a row's blocks follow one another."""
    scales = [0.5] * 4 + [0.5 * 2.0 ** -59.9, 0.5 * 2.0 ** -119.8]
    kv_heads, length = 200, 128 * len(scales)
    cache = Cache("int8", num_pages=len(scales), kv_heads=kv_heads, page_size=128, scale_block=128, head_dim=64, slots=1, max_pages=len(scales))
    cache.give_pages([length])
    cache.fill([length])
    cache.v.random_(60, 128, generator=cache.gen)
    for j, scale in enumerate(scales if falling else scales[::-1]):
        cache.vs[0, int(cache.table[0, j])] = scale
    q = (torch.randn((n, kv_heads, 64), generator=torch.Generator().manual_seed(6))).half()
    got = attend(gpu, liger, cache, [length], q, n, causal=0).double()
    want, mixed, size, top = attention(cache, 0, q, n, length, 0, 64 ** -0.5, 0)
    tol = attention_tolerance(want, mixed, size, 64) + lost_in_a_block(1.0, top)
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 7, 20, 60])
def test_blocks_whose_scale_one_key_has_set(gpu, liger, kind, d, n):
    """One key of a block has codes of -127 and so no weight, the few others are 0 but for codes of -1 and 1 here and there; all queries are positive and
    large.  A score is off by at most d * 2^-23 * sum |q code| of its own key, which is a thousandth of 128 * sum |q|."""
    lens = [3, 4, 6, 9]
    cache = Cache(kind, num_pages=8, kv_heads=1, page_size=16, scale_block=16, head_dim=d, slots=4, max_pages=2)
    cache.give_pages(lens)
    cache.fill(lens)
    codes = torch.randint(-1, 2, cache.k.shape, generator=cache.gen) * (torch.rand(cache.k.shape, generator=cache.gen) < 0.2)
    codes[:, :, :, 1] = -127 if kind == "int8" else -120
    cache.k = codes.to(torch.int8).view(torch.uint8) if kind == "int8" else codes.float().to(torch.float8_e4m3fn).view(torch.uint8)
    cache.ks.fill_(0.5)
    q = (60.0 + 8.0 * torch.randn((4 * n, 1, d), generator=torch.Generator().manual_seed(9))).half()
    scale = 1.0 / 64
    cache.to_gpu(liger)
    dq, dl = q.cuda(), ints(lens)
    out = torch.zeros((4 * n, d), dtype=torch.float16, device="cuda")
    a = attend_args(liger, cache, dq, out, dl, 1, n, 4, causal=0, scale=scale)
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    status(gpu)
    got = out.cpu().double().view(4, n, 1, d)
    for b, length in enumerate(lens):
        mine = q[b * n:(b + 1) * n]
        want, mixed, _, top = attention(cache, 0, mine, n, length, b, scale, 0)
        # the largest sum |q code| of the keys that weigh; the other one weighs less than 2^-100 however its score is rounded
        k = cache.values(0, b, length)[0][:, 0]
        k = k[k.abs().amax(-1) < 1.0]
        size = float((mine[:, 0].double().abs() @ k.abs().T).max()) * scale * 1.4427
        tol = attention_tolerance(want, mixed, size, d) + lost_in_a_block(1.0, top)
        off = (got[b] - want).abs()
        assert bool((off <= tol).all()), f"sequence {b}: worst {float((off / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [1, 20, 60])
def test_a_group_of_small_values_that_has_all_the_weight(gpu, liger, kind, n):
    """Inside one block of 128 keys: 16 keys weigh 2^30 times as much as the others and their values are 2^-20 of the others'."""
    length = 128
    cache = Cache(kind, num_pages=2, kv_heads=1, page_size=128, scale_block=16, head_dim=64, slots=1, max_pages=1)
    cache.give_pages([length])
    k, v = torch.randn((length, 1, 64), generator=cache.gen) * 0.2, 64.0 + 6.0 * torch.randn((length, 1, 64), generator=cache.gen)
    q = torch.randn((n, 1, 64), generator=torch.Generator().manual_seed(6)) * 0.2
    k[:, :, 0], q[:, :, 0] = 0.0, 4.0
    k[32:48, 0, 0] = 30 * 8 / (4.0 * 1.4427)
    cache.write(0, 0, k, v)
    cache.vs *= 512.0
    cache.vs[0, int(cache.table[0, 0]), 0, 2] *= 2.0 ** -20
    q = q.half()
    got = attend(gpu, liger, cache, [length], q, n, causal=0).double()
    want, mixed, size, top = attention(cache, 0, q, n, length, 0, 64 ** -0.5, 0)
    tol = attention_tolerance(want, mixed, size, 64) + lost_in_a_block(1.0, top)
    off = (got - want).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the tolerance, {float((off / want).max()):.3g} of the result"


@pytest.mark.parametrize("seed", range(8))
def test_calls_of_any_shape(gpu, liger, seed):
    """Types, pages, blocks, groups, lengths, runs, causal or not, scores from flat to a few keys that take all, value scales far apart: all within the
    bound of weights in two parts, with few rows and with many."""
    rng = random.Random(seed)
    for it in range(8):
        kind, d, page = rng.choice(["int8", "e4m3"]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256])
        block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
        kv_heads, group, batch = rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 5, 8, 13, 16, 20]), rng.randrange(1, 6)
        longest, most = rng.choice([40, 300, 1000, 3000 if it == 0 else 700]), rng.choice([1, 1, 3, 8, 40, 150])
        lens, many = [rng.randrange(0, longest + 1) for _ in range(batch)], [rng.randrange(0, most + 1) for _ in range(batch)]
        causal, amplify, spread = rng.choice([0, 1]), rng.choice([0.1, 1.0, 1.0, 4.0, 12.0, 30.0]), rng.choice([1.0, 30.0, 1e4])
        pages = -(-longest // page)
        cache = Cache(kind, num_pages=sum(-(-n // page) for n in lens) + 1, kv_heads=kv_heads, page_size=page, scale_block=block, head_dim=d, slots=batch,
                      max_pages=pages, seed=it)
        cache.give_pages(lens)
        cache.fill(lens, spread=spread)
        heads = kv_heads * group
        at = [sum(many[:b]) for b in range(batch + 1)]
        q = (torch.randn((at[-1] + 2, heads, d), generator=torch.Generator().manual_seed(it)) * amplify).half()
        got = attend(gpu, liger, cache, lens, q, max(max(many), 1), causal=causal, max_len=rng.choice([longest, pages * page]), offsets=at)
        assert bool((got[at[-1]:] == 7.0).all())
        for b, n in enumerate(many):
            want, mixed, size, top = attention(cache, 0, q[at[b]:at[b + 1]], n, lens[b], b, d ** -0.5, causal)
            tol = attention_tolerance(want, mixed, size, d) + lost_in_a_block(1.0, top)
            off = (got[at[b]:at[b + 1]].double() - want).abs()
            assert bool((off <= tol).all()), f"{it}: {kind} D{d} group {group} n {n} len {lens[b]} amplify {amplify}: {float((off / tol).max()):.3g} of the tolerance"
