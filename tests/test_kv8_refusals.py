"""liger_kv8_*: calls that the host refuses, before anything is launched (no GPU; the pointers are never dereferenced)."""
import ctypes as C

import pytest

OK, ODD = 0x7f0000001000, 0x7f0000001008  # 16-byte aligned / 8-byte aligned
INVALID, UNSUPPORTED, TOO_LARGE = -1, -3, -5


def cache(liger, **kw):
    c = liger.Kv8Cache()
    for n in ("k_pages", "v_pages", "k_scales", "v_scales", "page_table", "page_count", "page_refs"):
        setattr(c, n, OK)
    c.layers, c.num_pages, c.kv_heads, c.page_size, c.scale_block, c.head_dim, c.type, c.slots, c.max_pages = 2, 64, 4, 32, 16, 128, 0, 8, 16
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def append_args(liger, **kw):
    a = liger.Kv8AppendArgs()
    a.k, a.v, a.positions = OK, OK, OK
    a.batch, a.q_len, a.batch_stride, a.token_stride, a.head_stride = 4, 1, 512, 512, 128
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def attention_args(liger, **kw):
    a = liger.Kv8AttentionArgs()
    a.q, a.out, a.scratch, a.scratch_bytes, a.kv_lens = OK, OK, OK, 1 << 40, OK
    a.batch, a.heads, a.q_len, a.q_batch_stride, a.q_token_stride, a.q_head_stride = 4, 8, 1, 1024, 1024, 128
    a.max_kv_len, a.ldo, a.scale = 4096, 1024, 0.1
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD_CACHES = [(dict(k_pages=None), INVALID, "NULL"), (dict(v_scales=None), INVALID, "NULL"), (dict(page_table=None), INVALID, "NULL"),
              (dict(k_pages=ODD), INVALID, "aligned"), (dict(v_pages=ODD), INVALID, "aligned"), (dict(k_scales=OK + 2), INVALID, "aligned"),
              (dict(page_refs=OK + 2), INVALID, "aligned"), (dict(layers=0), INVALID, "positive"), (dict(num_pages=0), INVALID, "positive"),
              (dict(slots=-1), INVALID, "positive"), (dict(max_pages=0), INVALID, "positive"), (dict(kv_heads=0), INVALID, "positive"),
              (dict(head_dim=96), UNSUPPORTED, "head_dim"), (dict(type=2), INVALID, "type"), (dict(page_size=24), UNSUPPORTED, "page_size"),
              (dict(page_size=8), UNSUPPORTED, "page_size"), (dict(page_size=512), UNSUPPORTED, "page_size"),
              (dict(scale_block=64), UNSUPPORTED, "scale_block"), (dict(scale_block=8), UNSUPPORTED, "scale_block"),
              (dict(page_size=256, scale_block=256), UNSUPPORTED, "scale_block"), (dict(kv_heads=70000), UNSUPPORTED, "kv_heads"),
              (dict(max_pages=1 << 27), UNSUPPORTED, "max_pages"), (dict(num_pages=(1 << 30) + 1), UNSUPPORTED, "num_pages"),
              (dict(slots=(1 << 30) + 1), UNSUPPORTED, "slots")]


@pytest.mark.parametrize("kw,code,word", BAD_CACHES)
def test_bad_caches_are_refused_by_every_operator(liger, kw, code, word):
    lib, c = liger.lib(), cache(liger, **kw)
    by = C.byref(c)
    calls = [lambda: lib.liger_kv8_append(by, C.byref(append_args(liger)), None),
             lambda: lib.liger_kv8_attention(by, C.byref(attention_args(liger)), None),
             lambda: lib.liger_kv8_reserve(by, OK, OK, 4, OK, OK, 1 << 40, None),
             lambda: lib.liger_kv8_fork(by, OK, OK, OK, 4, OK, OK, 1 << 40, None),
             lambda: lib.liger_kv8_free(by, OK, 4, None),
             lambda: lib.liger_kv8_copy(by, OK, OK, 4, OK, OK, 1 << 40, None),
             lambda: lib.liger_kv8_compact(by, OK, OK, OK, 1 << 40, None)]
    for i, call in enumerate(calls):
        assert call() == code, i
        assert word in lib.liger_last_error().decode(), i
    assert lib.liger_kv8_attention_scratch_bytes(by, C.byref(attention_args(liger))) == 0


def test_a_missing_struct_is_refused(liger):
    lib, c = liger.lib(), cache(liger)
    assert lib.liger_kv8_append(None, C.byref(append_args(liger)), None) == INVALID
    assert lib.liger_kv8_append(C.byref(c), None, None) == INVALID
    assert lib.liger_kv8_attention(None, C.byref(attention_args(liger)), None) == INVALID
    assert lib.liger_kv8_attention(C.byref(c), None, None) == INVALID
    assert lib.liger_kv8_free(None, OK, 1, None) == INVALID
    assert lib.liger_kv8_pages_scratch_bytes(None, 1) == 0
    assert lib.liger_kv8_attention_scratch_bytes(None, None) == 0


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(positions=None), dict(k=ODD), dict(v=ODD), dict(positions=OK + 2),
                                dict(slots=OK + 1), dict(q_offsets=OK + 2), dict(batch=0), dict(q_len=0), dict(q_len=-4), dict(layer=2),
                                dict(layer=-1), dict(token_stride=4), dict(head_stride=12), dict(batch_stride=20), dict(token_stride=-512),
                                dict(q_offsets=OK, total_tokens=-1), dict(batch=60000, q_len=60000)])
def test_bad_append_arguments_are_refused(liger, kw):
    c = cache(liger)
    assert liger.lib().liger_kv8_append(C.byref(c), C.byref(append_args(liger, **kw)), None) == INVALID


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(kv_lens=None), dict(q=ODD), dict(out=ODD), dict(scratch=ODD),
                                dict(scratch=None), dict(kv_lens=OK + 2), dict(slots=OK + 2), dict(heads=6), dict(heads=0), dict(heads=-8),
                                dict(ldo=1016), dict(ldo=1028), dict(max_kv_len=-1), dict(layer=2), dict(layer=-1), dict(q_token_stride=1020),
                                dict(q_head_stride=-128), dict(q_batch_stride=1), dict(batch=0), dict(q_len=0),
                                dict(q_offsets=OK, total_tokens=-5)])
def test_bad_attention_arguments_are_refused(liger, kw):
    c = cache(liger)
    assert liger.lib().liger_kv8_attention(C.byref(c), C.byref(attention_args(liger, **kw)), None) == INVALID


def test_sizes_that_are_not_implemented_are_refused(liger):
    lib, c = liger.lib(), cache(liger)
    for kw in (dict(batch=70000), dict(q_len=(1 << 29) + 1, batch=1), dict(q_len=1 << 29, batch=1, heads=16)):
        a = attention_args(liger, ldo=4096, **kw)
        assert lib.liger_kv8_attention(C.byref(c), C.byref(a), None) == UNSUPPORTED
    assert lib.liger_kv8_append(C.byref(c), C.byref(append_args(liger, batch=70000)), None) == UNSUPPORTED


def test_page_operators_refuse_bad_arguments(liger):
    lib, c = liger.lib(), cache(liger)
    by, need = C.byref(c), lib.liger_kv8_pages_scratch_bytes(C.byref(c), 4)
    assert need > 0 and need % 16 == 0
    for bad in (dict(scratch=None), dict(scratch=ODD)):
        assert lib.liger_kv8_reserve(by, OK, OK, 4, OK, bad["scratch"], need, None) == INVALID
        assert lib.liger_kv8_fork(by, OK, OK, OK, 4, OK, bad["scratch"], need, None) == INVALID
        assert lib.liger_kv8_copy(by, OK, OK, 4, OK, bad["scratch"], need, None) == INVALID
        assert lib.liger_kv8_compact(by, OK, OK, bad["scratch"], need, None) == INVALID
    assert lib.liger_kv8_reserve(by, OK, OK, 4, OK, OK, need - 1, None) == TOO_LARGE
    assert lib.liger_kv8_fork(by, OK, OK, OK, 4, OK, OK, 0, None) == TOO_LARGE
    assert lib.liger_kv8_reserve(by, OK, OK, -1, OK, OK, need, None) == INVALID
    assert lib.liger_kv8_free(by, OK, -1, None) == INVALID
    assert lib.liger_kv8_free(by, OK, 0, None) == 0
    assert lib.liger_kv8_free(by, None, 2, None) == INVALID
    assert lib.liger_kv8_free(by, OK + 2, 2, None) == INVALID
    many = (1 << 28) + 1
    assert lib.liger_kv8_reserve(by, OK, OK, many, OK, OK, 1 << 40, None) == UNSUPPORTED
    assert lib.liger_kv8_fork(by, OK, OK, OK, many, OK, OK, 1 << 40, None) == UNSUPPORTED
    assert lib.liger_kv8_copy(by, OK, OK, many, OK, OK, 1 << 40, None) == UNSUPPORTED
    assert lib.liger_kv8_free(by, OK, many, None) == UNSUPPORTED
    assert lib.liger_kv8_pages_scratch_bytes(by, many) == 0
    for gone in ("page_count", "page_refs"):
        without = cache(liger, **{gone: None})
        assert lib.liger_kv8_free(C.byref(without), OK, 1, None) == INVALID
        assert lib.liger_kv8_reserve(C.byref(without), OK, OK, 4, OK, OK, need, None) == INVALID
        assert lib.liger_kv8_compact(C.byref(without), OK, OK, OK, need, None) == INVALID


def test_workspace_sizes_grow_with_what_they_are_for(liger):
    lib = liger.lib()
    small, big = cache(liger), cache(liger, num_pages=100000)
    assert lib.liger_kv8_pages_scratch_bytes(C.byref(big), 4) > lib.liger_kv8_pages_scratch_bytes(C.byref(small), 4)
    assert lib.liger_kv8_pages_scratch_bytes(C.byref(small), 1000) > lib.liger_kv8_pages_scratch_bytes(C.byref(small), 4)
    assert lib.liger_kv8_pages_scratch_bytes(C.byref(small), -1) == 0
    # attention: no call with smaller sizes needs more, so one workspace of the largest serves all
    def need(**kw):
        return lib.liger_kv8_attention_scratch_bytes(C.byref(wide), C.byref(attention_args(liger, ldo=1 << 20, **kw)))
    wide = cache(liger, page_size=256, max_pages=1 << 22)
    sizes = dict(batch=[1, 3, 40, 5000], q_len=[1, 2, 4, 5, 9, 16, 25, 100, 5000], max_kv_len=[0, 100, 1024, 1025, 100000, 1 << 24, (1 << 24) + 1, 1 << 30],
                 heads=[4, 8, 12, 48, 256])
    first = {n: v[1] for n, v in sizes.items()}
    for n, v in sizes.items():
        for other in sizes:
            for o in sizes[other]:
                got = [need(**{**first, other: o, n: x}) for x in v]
                assert got == sorted(got), (n, other, o)
    # the pointers in the arguments are not needed
    a = attention_args(liger, q=None, out=None, kv_lens=None, scratch=None)
    assert lib.liger_kv8_attention_scratch_bytes(C.byref(small), C.byref(a)) > 0
