"""The paged 8-bit key/value cache on the GPU, through the C ABI, against kv8_model (64-bit attention; codes, scales and page
tables exactly)."""
import ctypes as C

import pytest
import torch

from helpers import ptr, stream_ptr
from kv8_model import DTYPE, Cache, Pages, append, attention, attention_tolerance

pytestmark = pytest.mark.gpu
BAD_INDEX = 2


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def status(gpu, want=0):
    torch.cuda.synchronize()
    st = (C.c_uint * 4)()
    code = gpu.liger_device_status(C.byref(st))
    gpu.liger_device_status_clear()
    assert code == want, list(st)


def attend_args(liger, cache, q, out, lens, heads, q_len, batch, offsets=None, slots=None, total=0, strides=None, max_len=None,
                causal=1, layer=0, scale=None, ldo=None):
    a = liger.Kv8AttentionArgs()
    d = cache.head_dim
    a.q, a.out, a.kv_lens, a.batch, a.heads, a.q_len, a.total_tokens = q.data_ptr(), out.data_ptr(), lens.data_ptr(), batch, heads, q_len, total
    a.q_offsets = offsets.data_ptr() if offsets is not None else None
    a.slots = slots.data_ptr() if slots is not None else None
    a.q_batch_stride, a.q_token_stride, a.q_head_stride = strides or (q_len * heads * d, heads * d, d)
    a.max_kv_len = max(int(lens.max()), 0) if max_len is None else max_len
    a.ldo, a.layer, a.causal, a.scale = ldo or heads * d, layer, causal, d ** -0.5 if scale is None else scale
    size = liger.lib().liger_kv8_attention_scratch_bytes(cache.by, C.byref(a))
    a.keep = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")  # NaN: nothing is read that was not written
    a.scratch, a.scratch_bytes = a.keep.data_ptr(), size
    return a


def check_attention(got, cache, q, at, lens, slots, scale, causal, layer=0, what="", q_len=None):
    """`q_len`: the call's bound on new tokens; with more than 48 rows a key head the weights are single fp16 numbers."""
    heads, d = q.shape[1], q.shape[2]
    q_len = q_len or max(max(b - a for a, b in zip(at, at[1:])), 1)
    many_rows = q_len * (heads // cache.kv_heads) > 48
    for b, length in enumerate(lens):
        lo, hi = at[b], at[b + 1]
        want, mixed, size, top = attention(cache, layer, q[lo:hi], hi - lo, length, slots[b], scale, causal)
        off = (got[lo:hi].double().view(hi - lo, heads, d) - want).abs()
        tol = attention_tolerance(want, mixed, size, d, (length, top) if many_rows else None)
        assert bool((off <= tol).all()), f"{what} sequence {b} (n {hi - lo}, len {length}): worst {float((off / tol).max()):.3g} of the tolerance"


def run_attention(gpu, liger, cache, lens, many, heads, causal=1, slots=None, max_len=None, ragged=True, layer=0, seed=3, amplify=1.0):
    gen = torch.Generator().manual_seed(seed)
    d, batch = cache.head_dim, len(lens)
    at = [0]
    for n in many:
        at.append(at[-1] + n)
    rows = at[-1] + (2 if ragged else 0)
    q = (torch.randn((rows, heads, d), generator=gen) * amplify).half()
    out = torch.full((rows, heads * d), 7.0, dtype=torch.float16, device="cuda")
    cache.to_gpu(liger)
    a = attend_args(liger, cache, q.cuda(), out, ints(lens), heads, max(max(many), 1), batch, ints(at) if ragged else None,
                    ints(slots) if slots else None, rows, max_len=max_len, causal=causal, layer=layer)
    dq, dl, do, ds = q.cuda(), ints(lens), ints(at), ints(slots) if slots else None
    a.q, a.kv_lens = dq.data_ptr(), dl.data_ptr()
    a.q_offsets, a.slots = do.data_ptr() if ragged else None, ds.data_ptr() if slots else None
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    torch.cuda.synchronize()
    got = out.cpu()
    check_attention(got, cache, q, at, lens, slots or list(range(batch)), d ** -0.5, causal, layer, f"{cache.kind} D{d}")
    assert bool((got[at[-1]:] == 7.0).all()), "rows behind the last sequence were written"
    return got


# ---- attention ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (128, 128), (256, 32)])
def test_decode_lengths_around_every_border(gpu, liger, kind, d, page, block):
    """No token, one, and one more or less than a step, a block, a page."""
    lens = sorted({0, 1, 2, 15, 16, 17, block - 1, block + 1, page - 1, page, page + 1, 2 * page + 7})
    cache = Cache(kind, num_pages=sum(-(-n // page) for n in lens) + 2, kv_heads=3, page_size=page, scale_block=block, head_dim=d,
                  slots=len(lens), max_pages=4)
    cache.give_pages(lens)
    cache.fill(lens, spread=200.0)
    run_attention(gpu, liger, cache, lens, [1] * len(lens), heads=6, ragged=False)
    status(gpu)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 8, 9, 16, 20])
def test_decode_of_ragged_lengths_split_over_the_gpu(gpu, liger, kind, d, group):
    lens = [5000, 0, 37, 1600, 1, 2049, 700, 16]
    cache = Cache(kind, num_pages=330, kv_heads=2, page_size=32, scale_block=32, head_dim=d, slots=8, max_pages=160)
    cache.give_pages(lens)
    cache.fill(lens, spread=30.0)
    run_attention(gpu, liger, cache, lens, [1] * 8, heads=2 * group)
    status(gpu)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("max_len", [None, 100000])
def test_several_new_tokens_a_sequence(gpu, liger, d, causal, max_len):
    """Runs of new tokens, some longer than the sequence (their first rows see nothing), none, and ragged places."""
    lens, many = [300, 5, 0, 64, 33, 211], [5, 9, 3, 0, 33, 17]
    cache = Cache("int8", num_pages=60, kv_heads=2, page_size=16, scale_block=16, head_dim=d, slots=6, max_pages=7000)
    cache.give_pages(lens)
    cache.fill(lens)
    got = run_attention(gpu, liger, cache, lens, many, heads=6, causal=causal, max_len=max_len)
    if causal:
        assert bool((got[5:9] == 0).all()), "tokens in front of the sequence see nothing"
    assert bool((got[14:17] == 0).all()), "an empty sequence gives zeros"
    status(gpu)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("many,lens", [([130, 1, 257, 64], [130, 1, 700, 1000]), ([40, 300], [4100, 3000])])
def test_long_runs_of_new_tokens(gpu, liger, kind, d, causal, many, lens):
    cache = Cache(kind, num_pages=260, kv_heads=2, page_size=64, scale_block=32, head_dim=d, slots=4, max_pages=70)
    cache.give_pages(lens)
    cache.fill(lens, spread=40.0)
    run_attention(gpu, liger, cache, lens, many, heads=6, causal=causal)
    status(gpu)


def test_one_long_sequence_over_all_thread_blocks(gpu, liger):
    lens = [70001]
    cache = Cache("e4m3", num_pages=600, kv_heads=1, page_size=128, scale_block=64, head_dim=128, slots=1, max_pages=600)
    cache.give_pages(lens)
    cache.fill(lens)
    run_attention(gpu, liger, cache, lens, [1], heads=5)
    run_attention(gpu, liger, cache, lens, [40], heads=5)
    status(gpu)


def test_many_sequences_of_a_batch(gpu, liger):
    """More sequences than a thread block looks at in one round, most of them empty."""
    lens = [(i * 37) % 90 if i % 5 == 0 else 0 for i in range(700)]
    cache = Cache("int8", num_pages=900, kv_heads=1, page_size=16, scale_block=16, head_dim=64, slots=700, max_pages=64)
    cache.give_pages(lens)
    cache.fill(lens)
    run_attention(gpu, liger, cache, lens, [i % 3 for i in range(700)], heads=2, max_len=1000)
    status(gpu)


def test_slots_layers_and_shared_pages(gpu, liger):
    """Entries name slots in any order and the same one twice; the second layer is read."""
    lens = [100, 33, 250]
    cache = Cache("int8", layers=2, num_pages=40, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=3, max_pages=8)
    cache.give_pages(lens)
    cache.fill(lens, layer=1)
    run_attention(gpu, liger, cache, [250, 100, 250, 17], [1, 1, 2, 1], heads=4, slots=[2, 0, 2, 1], layer=1)
    status(gpu)


def test_queries_in_head_major_layout_and_wide_output_rows(gpu, liger):
    """q as LIGER_EPI_QKV_SPLIT writes it, [B, h, S, D]; output rows longer than heads * D keep what is behind."""
    B, h, S, d, lens = 2, 4, 5, 64, [40, 130]
    cache = Cache("e4m3", num_pages=20, kv_heads=4, page_size=16, scale_block=16, head_dim=d, slots=2, max_pages=9)
    cache.give_pages(lens)
    cache.fill(lens)
    cache.to_gpu(liger)
    q = torch.randn((B, h, S, d), generator=torch.Generator().manual_seed(1)).half()
    dq, dl = q.cuda(), ints(lens)
    out = torch.full((B * S, h * d + 24), 3.0, dtype=torch.float16, device="cuda")
    a = attend_args(liger, cache, dq, out, dl, h, S, B, strides=(h * S * d, d, S * d), ldo=h * d + 24)
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    torch.cuda.synchronize()
    rows = q.transpose(1, 2).reshape(B * S, h, d)
    check_attention(out[:, :h * d].cpu(), cache, rows, [0, S, 2 * S], lens, [0, 1], d ** -0.5, 1)
    assert bool((out[:, h * d:] == 3.0).all())
    status(gpu)


@pytest.mark.parametrize("many", [[1, 1], [3, 150]])
def test_zero_scales_large_scores_and_equal_keys(gpu, liger, many):
    lens = [200, 300]
    cache = Cache("int8", num_pages=12, kv_heads=1, page_size=64, scale_block=16, head_dim=64, slots=2, max_pages=5)
    cache.give_pages(lens)
    cache.fill(lens)
    page = int(cache.table[0, 1])
    cache.ks[0, page, 0, 1] = 0.0   # keys of zeros: scores 0
    cache.vs[0, page, 0, 2] = 0.0   # values of zeros
    cache.vs[0, int(cache.table[1, 0])] *= 1e4  # a block of much larger values
    cache.vs[0, int(cache.table[1, 2])] *= 1e-4
    run_attention(gpu, liger, cache, lens, many, heads=2, amplify=1.0)
    cache.fill(lens)
    run_attention(gpu, liger, cache, lens, many, heads=2, amplify=12.0)  # scores of about +-50: a few keys take all
    status(gpu)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("many", [1, 140])
@pytest.mark.parametrize("scales", [(1.0, 1e-40, 1e-30, 1.0, 3e-5, 1e-39), (1e-40, 0.0, 1e-41, 1e-30, 2e-7, 0.5), (0.0, 1e-40, 1e-45, 0.0, 1e-40, 1e-44),
                                    (40.0, 1e-12, 1e-20, 1e-25, 0.0, 1e-44)])
def test_value_scales_of_any_size_side_by_side(gpu, liger, kind, many, scales):
    """Finite scales that append does not write, numbers below the normal ones among them: a block whose values vanish beside another
    one's adds nothing, and its weights still count."""
    lens = [90, 37, 320, 16]
    cache = Cache(kind, num_pages=20, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=4, max_pages=16)
    cache.give_pages(lens)
    cache.fill(lens)
    for slot, n in enumerate(lens):
        for j in range(-(-n // 16)):
            cache.vs[0, int(cache.table[slot, j // 2]), :, j % 2] = scales[(j + slot) % len(scales)]
    run_attention(gpu, liger, cache, lens, [many] * 4, heads=4, ragged=False, max_len=5000)
    status(gpu)


def test_a_bound_on_the_lengths_far_above_them(gpu, liger):
    """Rows for the tensor-core kernel, in a cache that may grow to 2^29 tokens a sequence."""
    lens, many = [200, 0, 33], [60, 2, 40]
    cache = Cache("int8", num_pages=20, kv_heads=2, page_size=64, scale_block=16, head_dim=64, slots=3, max_pages=1 << 23)
    cache.give_pages(lens)
    cache.fill(lens)
    run_attention(gpu, liger, cache, lens, many, heads=4, max_len=1 << 29)
    status(gpu)


@pytest.mark.parametrize("many", [1, 140])
def test_values_that_are_not_finite_reach_only_those_who_see_them(gpu, liger, many):
    """A NaN block's rows are NaN; rows before it in causal order, other heads and other sequences are not."""
    lens = [200, 200]
    cache = Cache("e4m3", num_pages=12, kv_heads=2, page_size=64, scale_block=16, head_dim=64, slots=2, max_pages=5)
    cache.give_pages(lens)
    cache.fill(lens)
    cache.vs[0, int(cache.table[0, 2]), 1, 3] = float("inf")  # tokens 176 .. 191 of sequence 0, head 1
    cache.to_gpu(liger)
    q = torch.randn((2 * many, 2, 64), generator=torch.Generator().manual_seed(2)).half().cuda()
    out = torch.zeros((2 * many, 128), dtype=torch.float16, device="cuda")
    dl = ints(lens)
    a = attend_args(liger, cache, q, out, dl, 2, many, 2)
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    torch.cuda.synchronize()
    bad = out.isnan().view(2, many, 2, 64).cpu()
    first = 176 - (200 - many)  # the first row that sees them
    assert bool(bad[0, max(first, 0):, 1].all())
    assert not bool(bad[0, :max(first, 0)].any()) and not bool(bad[0, :, 0].any()) and not bool(bad[1].any())
    status(gpu)


@pytest.mark.parametrize("group", [1, 4, 6, 13, 20, 60])
def test_a_block_that_is_not_finite_inside_a_split_sequence(gpu, liger, group):
    """Its parts are joined inside a thread block and between thread blocks: the one head that sees it is NaN, the rest is right."""
    lens = [9000, 8000, 500]
    cache = Cache("int8", num_pages=280, kv_heads=2, page_size=64, scale_block=32, head_dim=128, slots=3, max_pages=160)
    cache.give_pages(lens)
    cache.fill(lens, spread=50.0)
    cache.ks[0, int(cache.table[0, 70]), 1, 1] = float("nan")
    cache.to_gpu(liger)
    heads = 2 * group
    q = torch.randn((3, heads, 128), generator=torch.Generator().manual_seed(8)).half()
    dq, dl = q.cuda(), ints(lens)
    out = torch.zeros((3, heads * 128), dtype=torch.float16, device="cuda")
    a = attend_args(liger, cache, dq, out, dl, heads, 1, 3)
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    torch.cuda.synchronize()
    got = out.cpu().view(3, heads, 128)
    assert bool(got[0, group:].isnan().all()) and not bool(got[0, :group].isnan().any()) and not bool(got[1:].isnan().any())
    cache.ks[0, int(cache.table[0, 70]), 1, 1] = 0.01  # the other head of sequence 0, and the other sequences
    got[0, group:] = attention(cache, 0, q[:1], 1, lens[0], 0, 128 ** -0.5, 1)[0][0, group:].half()
    check_attention(got.view(3, -1), cache, q, [0, 1, 2, 3], lens, [0, 1, 2], 128 ** -0.5, 1)
    status(gpu)


@pytest.mark.parametrize("many,group", [(1, 1), (1, 12), (3, 20)])
def test_bad_tables_lengths_and_offsets_are_left_out(gpu, liger, many, group):
    """Numbers on the device that name nothing: the kernels leave them out, say so, and answer the rest of the call."""
    lens = [90, 200, 64, 33]
    cache = Cache("int8", num_pages=20, kv_heads=1, page_size=32, scale_block=32, head_dim=64, slots=4, max_pages=7)
    cache.give_pages(lens)
    cache.fill(lens)
    cache.to_gpu(liger)
    q = torch.randn((4 * many, group, 64), generator=torch.Generator().manual_seed(5)).half()
    for kind in ("page", "negative page", "length", "too long", "slot"):
        table, told, slots = cache.table.clone(), list(lens), [0, 1, 2, 3]
        want_lens = list(lens)
        if kind == "page":
            table[1, 6] = 20          # tokens 192 .. 199 of sequence 1
        elif kind == "negative page":
            table[1, 6] = -1
        elif kind == "length":
            told[1], want_lens[1] = -3, 0
        elif kind == "too long":
            told[1], want_lens[1] = 7 * 32 + 1, 0
        else:
            slots[1], want_lens[1] = 4, 0
        cache.dev["table"].copy_(table)
        out = torch.full((4 * many, group * 64), 7.0, dtype=torch.float16, device="cuda")
        dq, dl, ds = q.cuda(), ints(told), ints(slots)
        for max_len in (300, 5000):
            a = attend_args(liger, cache, dq, out, dl, group, many, 4, slots=ds, max_len=max_len)
            if "page" in kind:
                a.causal = 0
            liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
            status(gpu, BAD_INDEX)
            if "page" in kind:   # as if the sequence ended before that page
                want_lens[1] = 192
            for b in range(4):
                check_attention(out.cpu()[b * many:(b + 1) * many], cache, q[b * many:(b + 1) * many], [0, many], [want_lens[b]], [b],
                                64 ** -0.5, a.causal, what=f"{kind} {b}")
    cache.dev["table"].copy_(cache.table)
    # offsets that are no runs of rows inside the call: those sequences bring nothing, the others are answered
    at = [0, many, 1, 4 * many + 9, 4 * many]
    out = torch.full((4 * many, group * 64), 7.0, dtype=torch.float16, device="cuda")
    dq, dl, do = q.cuda(), ints(lens), ints(at)
    a = attend_args(liger, cache, dq, out, dl, group, many, 4, offsets=do, total=4 * many)
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    status(gpu, BAD_INDEX)
    check_attention(out[:many].cpu(), cache, q[:many], [0, many], lens[:1], [0], 64 ** -0.5, 1)
    assert bool((out[many:] == 7.0).all())


def test_offsets_past_32_bits(gpu, liger):
    """Pages that begin more than 2^32 bytes into the pool."""
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GB")
    pages, page, d = 2600, 256, 128   # 2600 * 64 heads * 256 * 128 bytes = 5.4e9
    codes = torch.zeros((1, pages, 64, page, d), dtype=torch.int8, device="cuda")
    small = Cache("int8", num_pages=2, kv_heads=64, page_size=page, scale_block=32, head_dim=d, slots=1, max_pages=2)
    small.give_pages([300])
    small.fill([300])
    at = [pages - 1, pages - 2]
    values = codes.clone()
    scales = [torch.zeros((1, pages, 64, 8), device="cuda") for _ in range(2)]
    for i, p in enumerate(at):
        src = int(small.table[0, i])
        codes[0, p], values[0, p] = small.k[0, src].view(torch.int8).cuda(), small.v[0, src].view(torch.int8).cuda()
        scales[0][0, p], scales[1][0, p] = small.ks[0, src].cuda(), small.vs[0, src].cuda()
    table = ints([at])
    small.num_pages = pages
    small.c = small.struct(liger, dict(k=codes.data_ptr(), v=values.data_ptr(), ks=scales[0].data_ptr(), vs=scales[1].data_ptr(),
                                       table=table.data_ptr(), count=None, refs=None))
    small.num_pages = 2
    for many in (1, 40):
        q = torch.randn((many, 64, d), generator=torch.Generator().manual_seed(8)).half()
        out = torch.zeros((many, 64 * d), dtype=torch.float16, device="cuda")
        dq, dl = q.cuda(), ints([299])
        a = attend_args(liger, small, dq, out, dl, 64, many, 1)
        liger.check(gpu.liger_kv8_attention(small.by, C.byref(a), stream_ptr()))
        torch.cuda.synchronize()
        check_attention(out.cpu(), small, q, [0, many], [299], [0], d ** -0.5, 1)
    # and a token is written there
    k = torch.randn((1, 64, d), generator=torch.Generator().manual_seed(9)).half()
    b = liger.Kv8AppendArgs()
    dk, first = k.cuda(), ints([299])
    b.k, b.v, b.positions, b.batch, b.q_len = dk.data_ptr(), dk.data_ptr(), first.data_ptr(), 1, 1
    b.batch_stride, b.token_stride, b.head_stride = 64 * d, 64 * d, d
    liger.check(gpu.liger_kv8_append(small.by, C.byref(b), stream_ptr()))
    status(gpu)
    append(small, 0, 0, 299, k, k)
    assert torch.equal(codes[0, pages - 2].cpu(), small.k[0, int(small.table[0, 1])].view(torch.int8))


def test_two_streams_and_two_graphs_with_workspaces_of_their_own(gpu, liger):
    lens = [3000, 1234]
    cache = Cache("int8", num_pages=80, kv_heads=2, page_size=64, scale_block=16, head_dim=128, slots=2, max_pages=50)
    cache.give_pages(lens)
    cache.fill(lens)
    cache.to_gpu(liger)
    dl = ints(lens)
    q = [torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(i)).half() for i in range(2)]
    dq = [x.cuda() for x in q]
    out = [torch.zeros((2, 1024), dtype=torch.float16, device="cuda") for _ in range(2)]
    args = [attend_args(liger, cache, dq[i], out[i], dl, 8, 1, 2) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            liger.check(gpu.liger_kv8_attention(cache.by, C.byref(args[i]), C.c_void_p(streams[i].cuda_stream)))
    torch.cuda.synchronize()
    for i in range(2):
        check_attention(out[i].cpu(), cache, q[i], [0, 1, 2], lens, [0, 1], 128 ** -0.5, 1)
    first = [o.clone() for o in out]
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            liger.check(gpu.liger_kv8_attention(cache.by, C.byref(args[i]), stream_ptr()))
        graphs.append(g)
    dl.copy_(ints([2999, 77]))  # a replay reads the lengths of its time
    for o in out:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        check_attention(out[i].cpu(), cache, q[i], [0, 1, 2], [2999, 77], [0, 1], 128 ** -0.5, 1)
        assert not torch.equal(out[i], first[i])
    status(gpu)


def test_the_same_call_gives_the_same_bits(gpu, liger):
    lens = [9000, 50, 4000]
    cache = Cache("e4m3", num_pages=220, kv_heads=2, page_size=64, scale_block=64, head_dim=128, slots=3, max_pages=150)
    cache.give_pages(lens)
    cache.fill(lens)
    for many in ([1, 1, 1], [40, 1, 30]):
        a = run_attention(gpu, liger, cache, lens, many, heads=8)
        b = run_attention(gpu, liger, cache, lens, many, heads=8)
        assert torch.equal(a, b)


def test_scratch_that_is_too_small_is_refused(gpu, liger):
    cache = Cache("int8", num_pages=80, kv_heads=1, page_size=64, head_dim=64, slots=1, max_pages=40)
    cache.to_gpu(liger)
    q = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    dl = ints([0])
    a = attend_args(liger, cache, q, q, dl, 1, 1, 1, max_len=2000)
    assert a.scratch_bytes > 0
    a.scratch_bytes -= 1
    assert gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()) == -5
    assert b"needed" in gpu.liger_last_error()


# ---- append ------------------------------------------------------------------------------------------------------------------

def run_append(gpu, liger, cache, first, many, layer=0, slots=None, amplify=None, seed=4, ragged=True, k=None, v=None, skip=()):
    """Appends on both sides and compares the whole cache, bit for bit."""
    gen = torch.Generator().manual_seed(seed)
    at = [0]
    for n in many:
        at.append(at[-1] + n)
    shape = (at[-1], cache.kv_heads, cache.head_dim)
    k = torch.randn(shape, generator=gen).half() if k is None else k
    v = torch.randn(shape, generator=gen).half() if v is None else v
    if amplify:
        k, v = (k * amplify).half(), (v * amplify).half()
    a = liger.Kv8AppendArgs()
    dk, dv, do, dp = k.cuda(), v.cuda(), ints(at), ints(first)
    ds = ints(slots) if slots else None
    a.k, a.v, a.positions, a.batch, a.q_len, a.total_tokens, a.layer = dk.data_ptr(), dv.data_ptr(), dp.data_ptr(), len(many), max(max(many), 1), at[-1], layer
    a.q_offsets, a.slots = do.data_ptr() if ragged else None, ds.data_ptr() if slots else None
    row = cache.kv_heads * cache.head_dim
    a.batch_stride, a.token_stride, a.head_stride = a.q_len * row, row, cache.head_dim
    liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
    torch.cuda.synchronize()
    for b, n in enumerate(many):
        if b not in skip:
            append(cache, layer, (slots or range(len(many)))[b], first[b], k[at[b]:at[b + 1]], v[at[b]:at[b + 1]])
    same_cache(cache)


def same_cache(cache):
    got = cache.from_gpu()
    for n in ("ks", "vs"):
        want = getattr(cache, n)
        assert bool(((got[n] == want) | (got[n].isnan() & want.isnan())).all()), n
    for n in ("k", "v"):
        want = getattr(cache, n)
        same = got[n] == want
        if cache.kind == "e4m3":  # a zero may have either sign
            same |= ((got[n] & 0x7f) == 0) & ((want & 0x7f) == 0)
        assert bool(same.all()), f"{n}: {int((~same).sum())} codes differ, first at {(~same).nonzero()[0].tolist()}"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 32), (64, 64), (256, 128)])
def test_append_at_every_border_and_again_behind(gpu, liger, kind, d, page, block):
    """Runs that begin and end inside blocks and pages, then a few single tokens of growing size behind them: held codes are
    rounded again when a block's scale grows."""
    first = [0, 1, block - 1, block, page - 1, page + 3]
    many = [page + 5, block, 1, 2 * block + 1, 2, 0]
    cache = Cache(kind, layers=2, num_pages=26, kv_heads=3, page_size=page, scale_block=block, head_dim=d, slots=6, max_pages=6)
    cache.give_pages([4 * page] * 6)
    cache.fill([f for f in first], layer=1)
    cache.to_gpu(liger)
    run_append(gpu, liger, cache, first, many, layer=1)
    at = [f + n for f, n in zip(first, many)]
    for i in range(6):
        run_append(gpu, liger, cache, at, [1] * 6, layer=1, amplify=0.25 * 2 ** i, seed=20 + i, ragged=i % 2 == 0)
        at = [x + 1 for x in at]
    status(gpu)


def test_append_to_named_slots_once_each(gpu, liger):
    cache = Cache("int8", num_pages=20, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=4, max_pages=4)
    cache.give_pages([128] * 4)
    cache.fill([10, 20, 30, 40])
    cache.to_gpu(liger)
    run_append(gpu, liger, cache, [40, 10, 30], [3, 1, 20], slots=[3, 0, 2])
    status(gpu)
    run_append(gpu, liger, cache, [43, 11, 44, 50], [2, 1, 4, 1], slots=[3, 0, 3, 2], skip=(2,), seed=6)  # slot 3 twice
    status(gpu, BAD_INDEX)


def test_append_of_zeros_tiny_largest_and_not_finite_values(gpu, liger):
    for kind in ("int8", "e4m3"):
        cache = Cache(kind, num_pages=12, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=6, max_pages=2)
        cache.give_pages([64] * 6)
        cache.fill([8] * 6)
        cache.to_gpu(liger)
        k = torch.randn((6 * 20, 2, 64), generator=torch.Generator().manual_seed(1)).half()
        v = k.flip(0).contiguous()
        k[0:20] = 0.0
        v[20:40] = 6e-8          # the smallest fp16 number
        k[40:60] *= 60000 / k[40:60].abs().max()
        v[45, 0, 3] = 65504.0
        k[62, 1, 5] = float("inf")
        v[83, 0, 0] = float("nan")
        k[100:120] = -k[100:120].abs()
        run_append(gpu, liger, cache, [8] * 6, [20] * 6, k=k, v=v)
        run_append(gpu, liger, cache, [28] * 6, [3] * 6, seed=3)  # behind them, in the same blocks
        status(gpu)


def test_append_leaves_out_what_does_not_exist(gpu, liger):
    cache = Cache("e4m3", num_pages=12, kv_heads=2, page_size=32, scale_block=32, head_dim=64, slots=3, max_pages=3)
    cache.give_pages([96, 64, 64])
    cache.fill([5, 5, 5])
    cache.to_gpu(liger)
    cache.dev["table"][0, 1] = 12
    keep = {n: getattr(cache, n).clone() for n in ("k", "v", "ks", "vs")}
    page = int(cache.table[0, 1])
    k = torch.randn((64, 2, 64), generator=torch.Generator().manual_seed(3)).half()
    a = liger.Kv8AppendArgs()
    dk = k.cuda()
    a.k, a.v, a.batch, a.q_len = dk.data_ptr(), dk.data_ptr(), 1, 64
    a.batch_stride, a.token_stride, a.head_stride = 64 * 128, 128, 64

    def call(first, slots=None, offsets=None, total=0):
        hold = ints(first), ints(slots) if slots else None, ints(offsets) if offsets else None
        a.positions, a.slots, a.q_offsets, a.total_tokens = (hold[0].data_ptr(), *(t.data_ptr() if t is not None else None for t in hold[1:]), total)
        liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
        status(gpu, BAD_INDEX)

    call([5])  # page 1 of slot 0 does not exist: tokens 32 .. 63 are left out
    append(cache, 0, 0, 5, k, k)
    for n in keep:
        getattr(cache, n)[0, page] = keep[n][0, page]
    same_cache(cache)
    for bad in (dict(first=[-1]), dict(first=[33]), dict(first=[5], slots=[3]), dict(first=[5], slots=[-1]),
                dict(first=[5], offsets=[0, 65], total=64), dict(first=[5], offsets=[3, 2], total=64), dict(first=[5], offsets=[-1, 2], total=64)):
        call(**bad)
        same_cache(cache)


def test_append_takes_the_projection_s_layout(gpu, liger):
    """[B, h, S, D], as LIGER_EPI_QKV_SPLIT writes keys and values."""
    B, h, S, d = 2, 3, 21, 128
    cache = Cache("int8", num_pages=8, kv_heads=h, page_size=32, scale_block=32, head_dim=d, slots=2, max_pages=3)
    cache.give_pages([90, 90])
    cache.fill([6, 40])
    cache.to_gpu(liger)
    k, v = (torch.randn((B, h, S, d), generator=torch.Generator().manual_seed(i)).half() for i in range(2))
    dk, dv, first = k.cuda(), v.cuda(), ints([6, 40])
    a = liger.Kv8AppendArgs()
    a.k, a.v, a.positions, a.batch, a.q_len = dk.data_ptr(), dv.data_ptr(), first.data_ptr(), B, S
    a.batch_stride, a.token_stride, a.head_stride = h * S * d, d, S * d
    liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
    status(gpu)
    for b in range(B):
        append(cache, 0, b, [6, 40][b], k[b].transpose(0, 1), v[b].transpose(0, 1))
    same_cache(cache)


# ---- pages -------------------------------------------------------------------------------------------------------------------

class PagesOnGpu:
    """A cache whose page operators run on the GPU and on plain lists side by side."""

    def __init__(self, gpu, liger, num_pages=50, slots=7, max_pages=9, page_size=16, **kw):
        self.gpu, self.liger = gpu, liger
        self.cache = Cache(num_pages=num_pages, slots=slots, max_pages=max_pages, page_size=page_size, garbage=False, **kw)
        c = self.cache
        c.k.random_(0, 256, generator=c.gen)
        c.v.random_(0, 256, generator=c.gen)
        c.ks.normal_(generator=c.gen)
        c.vs.normal_(generator=c.gen)
        c.to_gpu(liger)
        self.model = Pages(num_pages, slots, max_pages, page_size)

    def scratch(self, n):
        size = self.gpu.liger_kv8_pages_scratch_bytes(self.cache.by, n)
        self.space = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        return ptr(self.space), size

    def moved(self, moves):
        for name in ("k", "v", "ks", "vs"):
            t = getattr(self.cache, name)
            old = t.clone()
            for a, b in moves:
                t[:, b] = old[:, a]

    def same(self):
        torch.cuda.synchronize()
        got = self.cache.from_gpu()
        table, count, refs = self.model.arrays()
        assert torch.equal(got["count"], count) and torch.equal(got["refs"], refs) and torch.equal(got["table"], table)
        for n in ("k", "v", "ks", "vs"):
            assert torch.equal(got[n], getattr(self.cache, n)), n

    def reserve(self, slots, lens):
        done, s, n = ints([-7] * len(slots)), ints(slots), ints(lens)
        self.liger.check(self.gpu.liger_kv8_reserve(self.cache.by, ptr(s), ptr(n), len(slots), ptr(done), *self.scratch(len(slots)), stream_ptr()))
        assert done.tolist() == self.model.reserve(slots, lens)
        self.same()

    def fork(self, src, dst, lens):
        done, s, d, n = ints([-7] * len(src)), ints(src), ints(dst), ints(lens)
        self.liger.check(self.gpu.liger_kv8_fork(self.cache.by, ptr(s), ptr(d), ptr(n), len(src), ptr(done), *self.scratch(len(src)), stream_ptr()))
        want, moves = self.model.fork(src, dst, lens)
        assert done.tolist() == want
        self.moved(moves)
        self.same()

    def free(self, slots):
        s = ints(slots)
        self.liger.check(self.gpu.liger_kv8_free(self.cache.by, ptr(s), len(slots), stream_ptr()))
        self.model.free(slots)
        self.same()

    def copy(self, src, dst):
        done, s, d = ints([-7] * len(src)), ints(src), ints(dst)
        self.liger.check(self.gpu.liger_kv8_copy(self.cache.by, ptr(s), ptr(d), len(src), ptr(done), *self.scratch(len(src)), stream_ptr()))
        want, moves = self.model.copy(src, dst)
        assert done.tolist() == want
        self.moved(moves)
        self.same()

    def compact(self):
        live, to = ints([-7]), ints([-7] * self.cache.num_pages)
        self.liger.check(self.gpu.liger_kv8_compact(self.cache.by, ptr(live), ptr(to), *self.scratch(0), stream_ptr()))
        n, want, moves = self.model.compact()
        assert live.item() == n and to.tolist() == want
        self.moved(moves)
        self.same()


@pytest.mark.parametrize("kw", [dict(), dict(kind="e4m3", layers=3, kv_heads=3, head_dim=128, page_size=32, scale_block=16),
                                dict(page_size=256, scale_block=64, kv_heads=5, head_dim=128)])
def test_pages_reserved_forked_freed_and_compacted(gpu, liger, kw):
    p = PagesOnGpu(gpu, liger, **kw)
    ps = p.cache.page_size
    p.reserve([2, 0, 5], [3 * ps, 1, 0])
    p.reserve([2, 0, 2, 6], [3 * ps + 1, ps, 9 * ps, 2 * ps - 1])       # slot 2 twice: the second entry is refused
    p.fork([2, 2, 0], [1, 3, 4], [2 * ps + 3, 3 * ps, 1])               # a part page, none, the only page
    p.fork([2, 6, 1, 6], [1, 5, 5, 0], [1, ps, 1, 1])                   # full slot, good, named before, full slot
    p.free([2, 3, 2])                                                   # twice: once
    p.compact()
    p.compact()
    p.reserve([2], [9 * ps])
    p.reserve([3], [9 * ps + 1])                                        # more than a table row has
    p.free([0, 1, 2, 3, 4, 5, 6])
    assert sum(p.model.refs) == 0
    p.compact()
    status(gpu)


def test_pages_run_out(gpu, liger):
    p = PagesOnGpu(gpu, liger, num_pages=10)
    p.reserve([0, 1, 2, 3], [64, 64, 64, 0])      # 4, 4, then 2 are left for 4; an entry that wants none is served
    p.fork([0, 0, 1, 0], [2, 3, 4, 5], [17, 33, 50, 16])   # two part pages are left for three; whole pages need none
    p.free([1])
    p.reserve([6], [16 * 9])
    p.reserve([6], [2 ** 31 - 1])
    status(gpu)


def test_page_operators_leave_out_what_does_not_exist(gpu, liger):
    p = PagesOnGpu(gpu, liger)
    p.reserve([0, 7, -1, 1], [40, 16, 16, 20])
    status(gpu, BAD_INDEX)
    p.reserve([2], [-5])
    status(gpu, BAD_INDEX)
    p.fork([0, 9, 0, -2, 0], [2, 3, 7, 4, 5], [33, 1, 1, 1, -1])
    status(gpu, BAD_INDEX)
    p.fork([0, 0, 1, 3], [0, 4, 5, 6], [1, 49, 33, 0])   # itself, longer than it is, longer, of an empty slot: nothing to hold
    status(gpu)
    p.free([3, 99, -1, 0])
    status(gpu, BAD_INDEX)
    p.copy([1, 50, 2, -1, 5], [3, 4, 50, 6, 7])
    status(gpu, BAD_INDEX)


def test_copies_with_targets_named_twice_and_chains(gpu, liger):
    p = PagesOnGpu(gpu, liger, layers=2, kv_heads=3, head_dim=128, page_size=64, scale_block=16)
    p.copy([1, 2, 3], [10, 11, 12])
    p.copy([1, 2, 4, 20], [20, 20, 5, 6])     # 20 twice; 20 is also a source
    p.copy([7, 8, 9, 9], [7, 9, 8, 30])       # onto itself; a swap is refused
    p.copy(list(range(25)), list(range(25, 50)))
    status(gpu)


def test_random_page_keeping(gpu, liger):
    import random
    rng = random.Random(11)
    p = PagesOnGpu(gpu, liger, num_pages=3000, slots=1500, max_pages=6, kv_heads=1, head_dim=64)
    slots = list(range(1500))
    for _ in range(4):
        p.reserve(rng.sample(slots, 1200), [rng.randrange(0, 90) for _ in range(1200)])
        empty = [s for s in slots if not p.model.table[s]] or [0]
        dst = [rng.choice(empty) for _ in range(300)]
        src = [rng.choice(slots) for _ in range(300)]
        p.fork(src, dst, [rng.randrange(0, 1 + 16 * len(p.model.table[s])) for s in src])
        p.free(rng.sample(slots, 700))
        p.compact()
    status(gpu)


# ---- together ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_serving_run(gpu, liger, kind):
    """Prompts of different lengths come in, tokens are generated, a sequence is forked and both branches go on, one ends, the
    pool is compacted, the rest goes on; every step's attention is checked against the cache as the model has it."""
    h, kvh, d, ps = 4, 2, 64, 16
    cache = Cache(kind, num_pages=40, kv_heads=kvh, page_size=ps, scale_block=16, head_dim=d, slots=4, max_pages=8)
    cache.to_gpu(liger)
    pages = Pages(40, 4, 8, ps)
    gen = torch.Generator().manual_seed(17)
    space = torch.empty(gpu.liger_kv8_pages_scratch_bytes(cache.by, 4), dtype=torch.uint8, device="cuda")
    length = {}

    def tables():
        cache.table, cache.count, cache.refs = pages.arrays()

    def step(slots, many):
        for s, n in zip(slots, many):
            length[s] = length.get(s, 0) + n
        ds, lens, first = ints(slots), ints([length[s] for s in slots]), ints([length[s] - n for s, n in zip(slots, many)])
        at = [0]
        for n in many:
            at.append(at[-1] + n)
        do = ints(at)
        liger.check(gpu.liger_kv8_reserve(cache.by, ptr(ds), ptr(lens), len(slots), None, ptr(space), space.numel(), stream_ptr()))
        pages.reserve(slots, [length[s] for s in slots])
        tables()
        k, v, q = (torch.randn((at[-1], n, d), generator=gen).half() for n in (kvh, kvh, h))
        dk, dv, dq = k.cuda(), v.cuda(), q.cuda()
        a = liger.Kv8AppendArgs()
        a.k, a.v, a.q_offsets, a.slots, a.positions = dk.data_ptr(), dv.data_ptr(), do.data_ptr(), ds.data_ptr(), first.data_ptr()
        a.token_stride, a.head_stride, a.batch, a.q_len, a.total_tokens = kvh * d, d, len(slots), max(many), at[-1]
        liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
        out = torch.zeros((at[-1], h * d), dtype=torch.float16, device="cuda")
        b = attend_args(liger, cache, dq, out, lens, h, max(many), len(slots), do, ds, at[-1], max_len=8 * ps)
        liger.check(gpu.liger_kv8_attention(cache.by, C.byref(b), stream_ptr()))
        torch.cuda.synchronize()
        for i, s in enumerate(slots):
            append(cache, 0, s, length[s] - many[i], k[at[i]:at[i + 1]], v[at[i]:at[i + 1]])
        same_cache(cache)
        check_attention(out.cpu(), cache, q, at, [length[s] for s in slots], slots, d ** -0.5, 1)

    step([0, 2, 1], [37, 5, 16])
    for _ in range(4):
        step([0, 1, 2], [1, 1, 1])
    ds, dd, dn = ints([0]), ints([3]), ints([length[0]])
    liger.check(gpu.liger_kv8_fork(cache.by, ptr(ds), ptr(dd), ptr(dn), 1, None, ptr(space), space.numel(), stream_ptr()))
    _, moves = pages.fork([0], [3], [length[0]])
    for a, b in moves:
        for t in (cache.k, cache.v, cache.ks, cache.vs):
            t[:, b] = t[:, a]
    tables()
    length[3] = length[0]
    step([3, 0, 1], [1, 1, 1])
    step([0, 3], [9, 2])
    gone = ints([1])
    liger.check(gpu.liger_kv8_free(cache.by, ptr(gone), 1, stream_ptr()))
    pages.free([1])
    liger.check(gpu.liger_kv8_compact(cache.by, None, None, ptr(space), space.numel(), stream_ptr()))
    _, _, moves = pages.compact()
    for t in (cache.k, cache.v, cache.ks, cache.vs):
        old = t.clone()
        for a, b in moves:
            t[:, b] = old[:, a]
    tables()
    length.pop(1)
    for _ in range(3):
        step([3, 2, 0], [1, 3, 1])
    got = cache.from_gpu()
    assert all(torch.equal(got[n], getattr(cache, n)) for n in ("table", "count", "refs"))
    status(gpu)


# ---- calls that padding, capturing and several streams make ---------------------------------------------------------------------

@pytest.mark.parametrize("group", [1, 40])
def test_a_call_in_which_nobody_brings_tokens(gpu, liger, group):
    """A batch of padding only: no rows, and nothing is written."""
    cache = Cache("int8", num_pages=20, kv_heads=2, page_size=16, head_dim=64, slots=3, max_pages=200)
    cache.give_pages([40, 0, 17])
    cache.fill([40, 0, 17])
    cache.to_gpu(liger)
    q = torch.zeros((1, 2 * group, 64), dtype=torch.float16, device="cuda")
    out = torch.full((1, 128 * group), 7.0, dtype=torch.float16, device="cuda")
    dl, do = ints([40, 0, 17]), ints([0, 0, 0, 0])
    for q_len in (1, 5):
        a = attend_args(liger, cache, q, out, dl, 2 * group, q_len, 3, offsets=do, total=0, max_len=3000)
        liger.check(gpu.liger_kv8_attention(cache.by, C.byref(a), stream_ptr()))
    b = liger.Kv8AppendArgs()
    b.k, b.v, b.q_offsets, b.positions, b.batch, b.q_len = q.data_ptr(), q.data_ptr(), do.data_ptr(), dl.data_ptr(), 3, 4
    b.token_stride, b.head_stride = 128, 64
    liger.check(gpu.liger_kv8_append(cache.by, C.byref(b), stream_ptr()))
    status(gpu)
    assert bool((out == 7.0).all())
    same_cache(cache)


def test_padding_entries_that_name_a_slot_in_use(gpu, liger):
    """Entries without tokens may name any slot, also one that a later entry writes to."""
    cache = Cache("e4m3", num_pages=12, kv_heads=2, page_size=32, scale_block=16, head_dim=64, slots=3, max_pages=4)
    cache.give_pages([96, 96, 96])
    cache.fill([20, 30, 40])
    cache.to_gpu(liger)
    run_append(gpu, liger, cache, [0, 20, 0, 30, 0], [0, 3, 0, 18, 0], slots=[0, 0, 1, 1, 1])
    status(gpu)


@pytest.mark.parametrize("q_len", [1, 60])
def test_a_captured_step_with_a_branch(gpu, liger, q_len):
    """reserve, append and attention captured behind work of another stream, replayed with other values in the same buffers."""
    h, d, ps = 2, 128, 32
    cache = Cache("int8", num_pages=40, kv_heads=h, page_size=ps, scale_block=32, head_dim=d, slots=2, max_pages=16)
    cache.to_gpu(liger)
    pages = Pages(40, 2, 16, ps)
    gen = torch.Generator().manual_seed(3)
    hk, hv, hq = (torch.randn((3, 2 * q_len, h, d), generator=gen).half() for _ in range(3))
    k, v, q = (x.cuda() for x in (hk, hv, hq))
    now_k, now_v, now_q = (torch.zeros_like(x[0]) for x in (k, v, q))
    lens, first, slots, step = ints([0, 0]), ints([0, 0]), ints([0, 1]), torch.zeros(1, dtype=torch.int64, device="cuda")
    out = torch.zeros((2 * q_len, h * d), dtype=torch.float16, device="cuda")
    space = torch.empty(gpu.liger_kv8_pages_scratch_bytes(cache.by, 2), dtype=torch.uint8, device="cuda")
    a = liger.Kv8AppendArgs()
    a.k, a.v, a.positions, a.batch, a.q_len = now_k.data_ptr(), now_v.data_ptr(), first.data_ptr(), 2, q_len
    a.batch_stride, a.token_stride, a.head_stride = q_len * h * d, h * d, d
    b = attend_args(liger, cache, now_q, out, lens, h, q_len, 2, max_len=500)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            now_q.copy_(q.index_select(0, step)[0])
        now_k.copy_(k.index_select(0, step)[0])
        now_v.copy_(v.index_select(0, step)[0])
        first.copy_(lens)
        lens.add_(q_len)
        liger.check(gpu.liger_kv8_reserve(cache.by, ptr(slots), ptr(lens), 2, None, ptr(space), space.numel(), stream_ptr()))
        liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
        main.wait_stream(side)
        liger.check(gpu.liger_kv8_attention(cache.by, C.byref(b), stream_ptr()))
        step.add_(1)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        length = (i + 1) * q_len
        pages.reserve([0, 1], [length, length])
        cache.table, cache.count, cache.refs = pages.arrays()
        for s in range(2):
            rows = slice(s * q_len, (s + 1) * q_len)
            append(cache, 0, s, i * q_len, hk[i, rows], hv[i, rows])
        same_cache(cache)
        check_attention(out.cpu(), cache, hq[i], [0, q_len, 2 * q_len], [length] * 2, [0, 1], d ** -0.5, 1, q_len=q_len)
    status(gpu)


def test_long_calls_on_two_streams_at_once(gpu, liger):
    lens = [2500, 700]
    cache = Cache("e4m3", num_pages=60, kv_heads=2, page_size=64, scale_block=32, head_dim=64, slots=2, max_pages=45)
    cache.give_pages(lens)
    cache.fill(lens)
    cache.to_gpu(liger)
    dl = ints(lens)
    q = [torch.randn((2 * 200, 4, 64), generator=torch.Generator().manual_seed(i)).half() for i in range(2)]
    dq = [x.cuda() for x in q]
    out = [torch.zeros((400, 256), dtype=torch.float16, device="cuda") for _ in range(2)]
    args = [attend_args(liger, cache, dq[i], out[i], dl, 4, 200, 2) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            liger.check(gpu.liger_kv8_attention(cache.by, C.byref(args[i]), C.c_void_p(streams[i].cuda_stream)))
    torch.cuda.synchronize()
    for i in range(2):
        check_attention(out[i].cpu(), cache, q[i], [0, 200, 400], lens, [0, 1], 64 ** -0.5, 1)
    status(gpu)


def test_projection_append_and_attention_in_a_row(gpu, liger):
    """The QKV projection's epilogue writes [B, h, 1, D]; its keys and values go into the cache and its queries look at it, as in a
    decode step, nothing waiting between."""
    B, h, d, H = 4, 3, 128, 256
    lens = [100, 7, 0, 63]
    cache = Cache("int8", num_pages=16, kv_heads=h, page_size=32, scale_block=16, head_dim=d, slots=B, max_pages=5)
    cache.give_pages([n + 1 for n in lens])
    cache.fill(lens)
    cache.to_gpu(liger)
    gen = torch.Generator().manual_seed(6)
    x, w = torch.randn((B, H), generator=gen).half().cuda(), (torch.randn((3 * h * d, H), generator=gen) * 0.06).half().cuda()
    q, k, v = (torch.zeros((B, h, 1, d), dtype=torch.float16, device="cuda") for _ in range(3))
    g = liger.GemmArgs()
    g.a, g.wt, g.q_out, g.k_out, g.v_out = x.data_ptr(), w.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr()
    g.m, g.n, g.k, g.lda, g.ldw, g.n_end, g.epilogue = B, 3 * h * d, H, H, H, 3 * h * d, liger.capi.EPI_QKV_SPLIT
    g.seq_len, g.heads, g.head_dim = 1, h, d
    first, after = ints(lens), ints([n + 1 for n in lens])
    out = torch.zeros((B, h * d), dtype=torch.float16, device="cuda")
    a = liger.Kv8AppendArgs()
    a.k, a.v, a.positions, a.batch, a.q_len = k.data_ptr(), v.data_ptr(), first.data_ptr(), B, 1
    a.batch_stride, a.token_stride, a.head_stride = h * d, d, d
    b = attend_args(liger, cache, q, out, after, h, 1, B, strides=(h * d, d, d))
    liger.check(gpu.liger_gemm_fp16(C.byref(g), stream_ptr()))
    liger.check(gpu.liger_kv8_append(cache.by, C.byref(a), stream_ptr()))
    liger.check(gpu.liger_kv8_attention(cache.by, C.byref(b), stream_ptr()))
    status(gpu)
    hq, hk, hv = (t.cpu()[:, :, 0] for t in (q, k, v))
    assert float(hk.abs().max()) > 0.5
    for s in range(B):
        append(cache, 0, s, lens[s], hk[s:s + 1], hv[s:s + 1])
    same_cache(cache)
    check_attention(out.cpu(), cache, hq, list(range(B + 1)), [n + 1 for n in lens], list(range(B)), d ** -0.5, 1)
