"""Operators of a paged key/value cache held in 8 bits: what is measured, in plain form and through the library.

The cache keeps, for every layer, pages of `page_size` tokens: codes [layers, pages, kv_heads, page_size, head_dim] in int8 or
e4m3, and one 32-bit scale for each block of `scale_block` tokens and head, [layers, pages, kv_heads, page_size / scale_block];
a value is code * scale.  A sequence is a row ("slot") of a page table.  Three operators work on it:

  attend   attention of new queries (one token a sequence, or a run of tokens) over the cache
  append   new keys and values are quantised and written behind the tokens that are there; where a block's scale has to grow,
           the tokens that it held are rounded again to the new one
  pages    keeping the pages: "branch" drops old branches of sequences, forks new ones and gives them room to grow,
           "compact" moves the pages in use to the front of the pool, "copy" copies pages onto others

`listed()` gives the cases that are timed, `draw()` more of the same ranges.
"""
import ctypes
import importlib
import math
import random

import torch

own = False

TYPES = {"int8": 0, "e4m3": 1}           # the library's numbers of the two types
QMAX = {"int8": 127.0, "e4m3": 448.0}    # the largest code


# ---- the cases -------------------------------------------------------------------------------------------------------------

def _attend(name, **kw):
    case = dict(op="attend", batch=1, q_len=1, ragged_q=False, kv_heads=8, group=1, head_dim=128, page_size=64, scale_block=16,
                type="int8", max_len=2048, lens="same", causal=True, pick=1)
    case.update(kw, name=name)
    return case


def _append(name, **kw):
    case = dict(op="append", batch=1, tokens=1, ragged_q=False, kv_heads=8, head_dim=128, page_size=64, scale_block=16, type="int8",
                max_len=2048, pick=1)
    case.update(kw, name=name)
    return case


def _pages(name, what, **kw):
    case = dict(op="pages", what=what, layers=4, num_pages=256, kv_heads=8, head_dim=128, page_size=16, scale_block=16, type="int8",
                slots=16, max_pages=64, count=8, pick=1)
    case.update(kw, name=name)
    return case


def listed():
    return [
        # one short conversation on a small model (16 heads of 64): a decode step's latency
        _attend("decode_one_short", batch=1, kv_heads=16, head_dim=64, page_size=16, max_len=133),
        # the decode benchmark's step: 32 sequences, 96 heads of 128, 2048 tokens each, plus the new one
        _attend("decode_batch32_mha", batch=32, kv_heads=96, page_size=64, scale_block=64, type="e4m3", max_len=2049),
        # continuous batching on a grouped-query model: lengths from none at all to many thousands
        _attend("decode_ragged_grouped", batch=48, kv_heads=8, group=8, page_size=32, max_len=16384, lens="spread", pick=3),
        # two long documents, few heads: rows must be split over the whole GPU
        _attend("decode_long_document", batch=2, kv_heads=4, group=5, page_size=128, scale_block=32, type="e4m3", max_len=150001, lens="near"),
        # checking a few drafted tokens a sequence against the cache
        _attend("verify_drafts", batch=12, q_len=5, ragged_q=True, kv_heads=8, group=4, page_size=16, max_len=6000, lens="behind", pick=5),
        # prompts of 512 tokens in chunks behind what was there already, 96 heads
        _attend("extend_prompts", batch=8, q_len=512, ragged_q=True, kv_heads=96, page_size=64, scale_block=32, max_len=2560, lens="behind", pick=7),
        # one token a sequence goes into the cache, a layer of the decode step on one of 8 ranks
        _append("append_one_each", batch=32, tokens=1, kv_heads=12, page_size=64, scale_block=16, type="e4m3", max_len=2049),
        # prompts of the benchmark's prefill go into the cache: 8 x 512 tokens, 96 heads, the first at odd places in their pages
        _append("append_prompts", batch=8, tokens=512, ragged_q=True, kv_heads=96, page_size=64, scale_block=32, max_len=1024, pick=2),
        # a few samples of one prompt are started again: small pages, little to copy
        _pages("branch_samples", "branch", num_pages=1000, slots=12, max_pages=60, count=8, layers=2),
        # a search with many beams, each round drops its old branches and forks from the kept ones
        _pages("branch_beams", "branch", num_pages=6000, slots=384, max_pages=64, count=256, kv_heads=12, page_size=32, type="e4m3", pick=2),
        # half of the sequences have ended: pages in use move to the front, so that the rest of the pool can be given back
        _pages("compact_pool", "compact", num_pages=2500, slots=64, max_pages=72, kv_heads=12, page_size=64, scale_block=32, pick=4),
        # pages of a prompt's prefix are copied for another group of sequences
        _pages("copy_prefix", "copy", num_pages=1600, kv_heads=12, page_size=64, scale_block=64, count=600, type="e4m3", pick=6),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: the kinds in turn of a die, sizes over their whole ranges, held below the largest listed case's work."""
    page = rng.choice((16, 32, 64, 128, 256))
    shape = dict(head_dim=rng.choice((64, 128)), page_size=page, scale_block=rng.choice([b for b in (16, 32, 64, 128) if b <= page]),
                 type=rng.choice(("int8", "e4m3")), pick=rng.randrange(1, 1 << 20))
    kind = rng.choice(("decode", "decode", "verify", "extend", "append", "append", "branch", "compact", "copy"))
    if kind in ("decode", "verify", "extend"):
        case = dict(_attend("", **shape), batch=_log(rng, 1, 64), kv_heads=rng.choice((1, 2, 3, 4, 8, 12, 16, 24, 32, 96)),
                    group=rng.choice((1, 1, 2, 3, 4, 5, 7, 8, 12, 16)), lens=rng.choice(("same", "near", "spread", "behind")), max_len=_log(rng, 1, 100000))
        if kind == "verify":
            case.update(q_len=rng.randrange(2, 17), ragged_q=rng.random() < 0.5)
        if kind == "extend":
            case.update(q_len=_log(rng, 17, 700), ragged_q=rng.random() < 0.7, causal=rng.random() < 0.8, max_len=_log(rng, 1, 6000))
        big = 1 << 29
        while (case["batch"] * case["kv_heads"] * case["max_len"] * case["head_dim"] * 2 > big
               or case["batch"] * case["kv_heads"] * case["group"] * case["q_len"] * case["max_len"] > (1 << 28)):
            at = rng.choice(("batch", "kv_heads", "max_len", "group"))
            case[at] = max(1, case[at] * 2 // 3)
    elif kind == "append":
        case = dict(_append("", **shape), batch=_log(rng, 1, 64), tokens=_log(rng, 1, 700), ragged_q=rng.random() < 0.6,
                    kv_heads=rng.choice((1, 2, 4, 8, 12, 16, 48)))
        while case["batch"] * case["tokens"] * case["kv_heads"] * case["head_dim"] > (1 << 25):
            case["batch"] = max(1, case["batch"] // 2)
            case["tokens"] = max(1, case["tokens"] * 2 // 3)
        case["max_len"] = case["tokens"] + _log(rng, 1, 1000)
    else:
        case = dict(_pages("", kind, **shape), layers=rng.randrange(1, 5), kv_heads=rng.choice((1, 2, 4, 8, 12)), slots=_log(rng, 3, 300),
                    max_pages=_log(rng, 2, 64))
        while case["slots"] * case["max_pages"] * _page_bytes(case) > (1 << 30):
            case["slots"] = max(3, case["slots"] // 2)
            case["max_pages"] = max(2, case["max_pages"] * 2 // 3)
        case["num_pages"] = case["slots"] * case["max_pages"] + rng.randrange(8, 200)
        case["count"] = _log(rng, 1, case["num_pages"] // 2) if kind == "copy" else rng.randrange(1, max(2, case["slots"] // 2))
    del case["name"]
    return case


def _page_bytes(case):
    """Bytes of one page in all layers: codes and scales, keys and values."""
    return 2 * case["layers"] * case["kv_heads"] * case["page_size"] * (case["head_dim"] + 4 / case["scale_block"])


def _lens(case):
    """Tokens of each sequence after this call: all alike, nearly alike, spread from none to the longest, or anything behind the new ones."""
    rng, top = random.Random(case["pick"]), case["max_len"]
    if case["lens"] == "same":
        return [top] * case["batch"]
    if case["lens"] == "near":
        return [top] + [max(1, top - rng.randrange(0, 1 + top // 50)) for _ in range(case["batch"] - 1)]
    if case["lens"] == "behind":
        return [top] + [rng.randrange(min(n, top), top + 1) for n in _new_tokens(case, case["q_len"])[1:]]
    lens = [min(top, int(top ** (0.4 + 0.6 * rng.random()))) for _ in range(case["batch"])]
    lens[0] = top
    if case["batch"] > 3:
        lens[2] = 0
    return lens


def _new_tokens(case, longest):
    """New tokens of each sequence: `longest`, or from none to `longest`."""
    rng = random.Random(case["pick"] + 1)
    if not case["ragged_q"]:
        return [longest] * case["batch"]
    many = [rng.randrange(0 if b % 5 == 3 else 1, longest + 1) for b in range(case["batch"])]
    many[0] = longest
    return many


def _append_places(case):
    """(new tokens, position of the first) of each sequence."""
    rng, many = random.Random(case["pick"] + 2), _new_tokens(case, case["tokens"])
    room = case["max_len"] - case["tokens"]
    return many, [0 if b % 7 == 5 else rng.randrange(room // 2, room + 1) for b in range(case["batch"])]


def work(case):
    d = case["head_dim"]
    if case["op"] == "attend":
        lens, many = _lens(case), _new_tokens(case, case["q_len"])
        heads = case["kv_heads"] * case["group"]
        seen = 0
        for n, l in zip(many, lens):
            first = l - n
            seen += sum(min(l, max(0, first + i + 1)) for i in range(n)) if case["causal"] else n * l
        tokens = sum(l for n, l in zip(many, lens) if n)
        return {"bytes": 2 * tokens * case["kv_heads"] * (d + 4 / case["scale_block"]) + 4 * sum(many) * heads * d, "flops": 4 * d * heads * seen}
    if case["op"] == "append":
        many, _ = _append_places(case)
        return {"bytes": 2 * sum(many) * case["kv_heads"] * (3 * d + 4 / case["scale_block"]), "flops": 4 * sum(many) * case["kv_heads"] * d}
    p = _bookkeeping(case)
    moved = len(p["moves"]) if case["what"] != "branch" else sum(1 for l in p["lens"] if l % case["page_size"])
    return {"bytes": 2 * moved * _page_bytes(case) + 4 * (2 * case["num_pages"] + case["slots"] * case["max_pages"]), "flops": 0}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _fill_pool(case, layers, pages, gen):
    """Codes and scales as quantising normal values gives them; pages that nothing was written to hold any bytes at all."""
    shape = (layers, pages, case["kv_heads"], case["page_size"], case["head_dim"])
    blocks = case["page_size"] // case["scale_block"]
    codes = torch.empty(shape, dtype=torch.int8 if case["type"] == "int8" else torch.float8_e4m3fn, device="cuda")
    flat = codes.view(torch.uint8).view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        piece = torch.randn(min(1 << 28, flat.numel() - at), generator=gen, device="cuda")
        if case["type"] == "int8":
            piece = piece.mul_(45).round_().clamp_(-127, 127).to(torch.int8)
        else:
            piece = piece.mul_(150).clamp_(-448, 448).to(torch.float8_e4m3fn)
        flat[at:at + piece.numel()] = piece.view(torch.uint8)
    scales = torch.rand((layers, pages, case["kv_heads"], blocks), generator=gen, device="cuda").mul_(0.8).add_(0.6).mul_(2.8 / QMAX[case["type"]])
    return codes, scales


def _tables(case, lens, gen, spare):
    """A page table whose pages lie anywhere in the pool, and its size."""
    per = max(1, -(-case["max_len"] // case["page_size"]))
    need = [-(-l // case["page_size"]) for l in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), per), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(many):
    at = [0]
    for n in many:
        at.append(at[-1] + n)
    return at


def _bookkeeping(case):
    """Where the pages are before the call, as plain numbers: the table, how often each page is used, and what is asked."""
    rng, ps, n = random.Random(case["pick"] + 3), case["page_size"], case["num_pages"]
    free, table, refs = list(range(n)), [[] for _ in range(case["slots"])], [0] * n
    if case["what"] == "copy":
        order = rng.sample(range(n), min(n // 2, case["count"]) * 2)
        return {"moves": list(zip(order[0::2], order[1::2])), "table": table, "refs": refs}
    rng.shuffle(free)
    if case["what"] == "compact":
        for s in range(case["slots"]):
            many = rng.randrange(0, case["max_pages"] + 1) if s % 2 else 0
            table[s] = [free.pop() for _ in range(min(many, len(free)))]
        for s in range(3, case["slots"], 4):  # some share the beginning of another
            share = table[s - 2][:len(table[s]) // 2]
            free += table[s][:len(share)]
            table[s][:len(share)] = share
        for row in table:
            for p in row:
                refs[p] += 1
        live = sum(r > 0 for r in refs)
        to = [p for p in range(live) if refs[p] == 0]
        return {"moves": list(zip((p for p in range(live, n) if refs[p]), to)), "table": table, "refs": refs}
    # branch: the first slots are kept sequences, the last `count` old branches of them
    kept = case["slots"] - case["count"]
    lens = [rng.randrange(1, max(2, ps * max(1, case["max_pages"] - 2))) for _ in range(kept)]
    room = max(1, (n - case["count"] * 4) // max(1, kept))
    lens = [min(l, room * ps) for l in lens]
    for s in range(kept):
        table[s] = [free.pop() for _ in range(-(-lens[s] // ps))]
    for s in range(kept, case["slots"]):
        of = rng.randrange(kept)
        table[s] = table[of][:lens[of] // ps] + [free.pop()]
    for row in table:
        for p in row:
            refs[p] += 1
    src = [rng.randrange(kept) for _ in range(case["count"])]
    return {"moves": [], "table": table, "refs": refs, "src": src, "dst": list(range(kept, case["slots"])),
            "lens": [lens[s] for s in src], "grown": [min(lens[s] + rng.randrange(1, 2 * ps), case["max_pages"] * ps) for s in src]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    d, kvh = case["head_dim"], case["kv_heads"]
    if case["op"] == "attend":
        lens, many = _lens(case), _new_tokens(case, case["q_len"])
        s["table"], pages = _tables(case, lens, gen, 3)
        s["k"], s["ks"] = _fill_pool(case, 1, pages, gen)
        s["v"], s["vs"] = _fill_pool(case, 1, pages, gen)
        at, heads = _offsets(many), kvh * case["group"]
        rows = at[-1] + (3 if case["ragged_q"] else 0)  # rows behind the last sequence stay as they are
        s["q"] = torch.randn((rows, heads, d), generator=gen, device="cuda").half()
        s["out"] = torch.full((rows, heads * d), 2.0 ** -6, dtype=torch.float16, device="cuda")
        s["lens"], s["offsets"] = _ints(lens), _ints(at)
        # where each new token stands in a padded batch, and the other way
        s["of_row"] = _ints([b for b, n in enumerate(many) for _ in range(n)]).long()
        s["in_row"] = _ints([i for n in many for i in range(n)]).long()
        s["many"], s["rows"] = _ints(many), at[-1]
        s["scale"] = d ** -0.5
    elif case["op"] == "append":
        many, first = _append_places(case)
        lens = [p + n for p, n in zip(first, many)]
        s["table"], pages = _tables(case, lens, gen, 2)
        s["k"], s["ks"] = _fill_pool(case, 1, pages, gen)
        s["v"], s["vs"] = _fill_pool(case, 1, pages, gen)
        at = _offsets(many)
        s["new_k"] = torch.randn((at[-1], kvh, d), generator=gen, device="cuda").mul_(1.1).half()
        s["new_v"] = torch.randn((at[-1], kvh, d), generator=gen, device="cuda").half()
        s["offsets"], s["first"] = _ints(at), _ints(first)
        s["of_row"] = _ints([b for b, n in enumerate(many) for _ in range(n)]).long()
        s["in_row"] = _ints([i for n in many for i in range(n)]).long()
        s["many"], s["rows"] = _ints(many), at[-1]
        s["rqmax"] = torch.tensor(1.0 / QMAX[case["type"]], dtype=torch.float32, device="cuda")
    else:
        p = _bookkeeping(case)
        s["k"], s["ks"] = _fill_pool(case, case["layers"], case["num_pages"], gen)
        s["v"], s["vs"] = _fill_pool(case, case["layers"], case["num_pages"], gen)
        width = case["max_pages"]
        s["table"] = _ints([row + [-1] * (width - len(row)) for row in p["table"]])
        s["held"], s["refs"] = _ints([len(row) for row in p["table"]]), _ints(p["refs"])
        s["before"] = s["table"].clone(), s["refs"].clone()
        s["done"] = torch.zeros(max(1, case["count"], len(p["moves"])), dtype=torch.int32, device="cuda")
        s["roomy"] = torch.zeros_like(s["done"])
        if case["what"] == "copy":
            s["src"], s["dst"] = _ints([m[0] for m in p["moves"]]), _ints([m[1] for m in p["moves"]])
        if case["what"] == "branch":
            for key in ("src", "dst", "lens", "grown"):
                s[key] = _ints(p[key])
        s["live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["moved_to"] = torch.zeros(case["num_pages"], dtype=torch.int32, device="cuda")
    return s


# ---- a pass ----------------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _through_library(s)
    what = s["case"]["op"]
    return _plain_attend(s) if what == "attend" else _plain_append(s) if what == "append" else _PLAIN_PAGES[s["case"]["what"]](s)


def _through_library(s):
    """The calls that a program makes; what it sets up once for these buffers (descriptors, workspace) is kept with them."""
    if "calls" not in s:
        s["calls"] = _set_up(s)
    if s["case"]["op"] == "pages" and s["case"]["what"] == "compact":
        s["table"].copy_(s["before"][0])
        s["refs"].copy_(s["before"][1])
    check, calls, answer = s["calls"]
    stream = torch.cuda.current_stream().cuda_stream
    for call, args in calls:
        check(call(*args, stream))
    return answer


def _set_up(s):
    """The library's descriptors for these buffers, the workspace, and what is called in order."""
    liger = importlib.import_module("24ppopp-liger_b200")
    lib, case = liger.lib(), s["case"]
    at = lambda t: t.data_ptr()  # noqa: E731
    cache = liger.Kv8Cache()
    cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales = at(s["k"]), at(s["v"]), at(s["ks"]), at(s["vs"])
    cache.layers, cache.num_pages, cache.kv_heads, cache.page_size, cache.head_dim = s["k"].shape
    cache.scale_block, cache.type = case["scale_block"], TYPES[case["type"]]
    cache.page_table, (cache.slots, cache.max_pages) = at(s["table"]), s["table"].shape
    by = ctypes.byref(cache)

    def workspace(size):
        s["scratch"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        return at(s["scratch"]), size

    if case["op"] == "attend":
        a = liger.Kv8AttentionArgs()
        heads, d = case["kv_heads"] * case["group"], case["head_dim"]
        a.q, a.out, a.kv_lens, a.batch, a.heads, a.q_len = at(s["q"]), at(s["out"]), at(s["lens"]), case["batch"], heads, case["q_len"]
        a.q_offsets, a.total_tokens = at(s["offsets"]) if case["ragged_q"] else None, s["q"].shape[0]
        a.q_batch_stride, a.q_token_stride, a.q_head_stride = case["q_len"] * heads * d, heads * d, d
        a.max_kv_len, a.ldo, a.layer, a.causal, a.scale = case["max_len"], heads * d, 0, int(case["causal"]), s["scale"]
        a.scratch, a.scratch_bytes = workspace(lib.liger_kv8_attention_scratch_bytes(by, ctypes.byref(a)))
        return liger.check, [(lib.liger_kv8_attention, (by, ctypes.byref(a)))], s["out"]
    if case["op"] == "append":
        a = liger.Kv8AppendArgs()
        a.k, a.v, a.positions, a.batch, a.q_len = at(s["new_k"]), at(s["new_v"]), at(s["first"]), case["batch"], case["tokens"]
        a.q_offsets, a.total_tokens = at(s["offsets"]) if case["ragged_q"] else None, s["new_k"].shape[0]
        row = case["kv_heads"] * case["head_dim"]
        a.batch_stride, a.token_stride, a.head_stride, a.layer = case["tokens"] * row, row, case["head_dim"], 0
        return liger.check, [(lib.liger_kv8_append, (by, ctypes.byref(a)))], _cache_of(s)
    cache.page_count, cache.page_refs = at(s["held"]), at(s["refs"])
    space = workspace(lib.liger_kv8_pages_scratch_bytes(by, s["done"].numel()))
    if case["what"] == "copy":
        calls = [(lib.liger_kv8_copy, (by, at(s["src"]), at(s["dst"]), s["src"].numel(), at(s["done"]), *space))]
    elif case["what"] == "compact":
        calls = [(lib.liger_kv8_compact, (by, at(s["live"]), at(s["moved_to"]), *space))]
    else:
        n = case["count"]
        calls = [(lib.liger_kv8_free, (by, at(s["dst"]), n)),
                 (lib.liger_kv8_fork, (by, at(s["src"]), at(s["dst"]), at(s["lens"]), n, at(s["done"]), *space)),
                 (lib.liger_kv8_reserve, (by, at(s["dst"]), at(s["grown"]), n, at(s["roomy"]), *space))]
    return liger.check, calls, _pages_answer(s)


def _cache_of(s):
    return {"k": s["k"], "v": s["v"], "k_scales": s["ks"], "v_scales": s["vs"]}


def _pages_answer(s):
    return {**_cache_of(s), "table": s["table"], "held": s["held"], "refs": s["refs"], "done": s["done"], "roomy": s["roomy"],
            "live": s["live"], "moved_to": s["moved_to"]}


# ---- plain forms -----------------------------------------------------------------------------------------------------------

def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _values(codes, scales, table):
    """What the cache holds for every sequence, [batch, kv_heads, tokens, head_dim] in 32 bits."""
    where = table.clamp(min=0).long()
    c = _bytes(codes)[0][where].view(codes.dtype).float()  # batch, page, head, token, dim
    b, p, h, t, d = c.shape
    c = c.view(b, p, h, scales.shape[-1], -1, d) * scales[0][where][..., None, None]
    return c.view(b, p, h, t, d).transpose(1, 2).reshape(b, h, p * t, d)


def _plain_attend(s):
    case = s["case"]
    b, n, kvh, g, d = case["batch"], case["q_len"], case["kv_heads"], case["group"], case["head_dim"]
    k, v = _values(s["k"], s["ks"], s["table"]), _values(s["v"], s["vs"], s["table"])
    keys = torch.arange(k.shape[2], device="cuda")
    there = (keys < s["lens"][:, None])[:, None, :, None]
    k, v = torch.where(there, k, 0.0), torch.where(there, v, 0.0)
    q = torch.zeros((b, n, kvh, g, d), device="cuda")
    q[s["of_row"], s["in_row"]] = s["q"][:s["rows"]].float().view(-1, kvh, g, d)
    x = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(b, kvh, n * g, d), k.transpose(2, 3)).mul_(s["scale"])
    # token i of m new ones stands at place len - m + i, and sees what is not behind it
    place = s["lens"][:, None] - s["many"][:, None] + torch.arange(n, device="cuda") if case["causal"] else (s["lens"] - 1)[:, None].expand(b, n)
    hidden = keys > torch.minimum(place, s["lens"][:, None] - 1)[..., None]  # batch, token, key
    x = x.view(b, kvh, n, g, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    x = torch.matmul(x.view(b, kvh, n * g, -1), v).view(b, kvh, n, g, d) / torch.where(total == 0, 1.0, total)
    s["out"][:s["rows"]] = x.permute(0, 2, 1, 3, 4)[s["of_row"], s["in_row"]].reshape(-1, kvh * g * d).half()
    return s["out"]


def _rounded(y, kind):
    top = QMAX["int8" if kind == torch.int8 else "e4m3"]
    y = y.round() if kind == torch.int8 else y
    return y.clamp(-top, top).to(kind)


def _plain_append_to(s, codes, scales, new):
    case = s["case"]
    ps, sb = case["page_size"], case["scale_block"]
    old_scales = scales[0].clone()
    place = s["first"].long()[s["of_row"]] + s["in_row"]
    page, inside = s["table"].long()[s["of_row"], place // ps], place % ps
    new = new.float()
    block = page * (ps // sb) + inside // sb
    pages, kvh, blocks = scales.shape[1:]
    most = torch.zeros((pages * blocks, kvh), device="cuda").index_reduce_(0, block, new.abs().amax(-1), "amax")
    wanted = (most * s["rqmax"]).view(pages, blocks, kvh).transpose(1, 2)
    touched = torch.zeros(pages * blocks, dtype=torch.bool, device="cuda").index_fill_(0, block, True).view(pages, 1, blocks)
    # the block that a sequence's first new token falls into keeps what it holds, at a scale that is no smaller
    who = torch.where(s["many"] > 0, torch.arange(case["batch"], device="cuda"), 0)  # who brings nothing repeats the first
    start = s["first"].long()[who]
    page_b, block_b = s["table"].long()[who, start // ps], start % ps // sb
    goes_on = (start % sb > 0).view(-1, 1)
    held = torch.zeros_like(old_scales)
    held[page_b, :, block_b] = torch.where(goes_on, old_scales[page_b, :, block_b], 0.0)
    scales[0] = torch.where(touched, torch.maximum(wanted, held), old_scales)
    back = torch.where(scales[0] > 0, 1.0 / scales[0], 0.0)
    # what the block holds is rounded to its new scale
    rows = block_b[:, None] * sb + torch.arange(sb, device="cuda")
    old = _bytes(codes)[0][page_b[:, None], :, rows]  # batch, token, head, dim
    ratio = old_scales[page_b, :, block_b] * back[page_b, :, block_b]
    again = _bytes(_rounded(old.view(codes.dtype).float() * ratio[:, None, :, None], codes.dtype))
    kept = goes_on & (rows < (start % ps)[:, None])
    flat = _bytes(codes)[0]
    flat[page_b[:, None], :, rows] = torch.where(kept[..., None, None], again, old)
    flat[page, :, inside] = _bytes(_rounded(new * back[page, :, inside // sb][..., None], codes.dtype))


def _plain_append(s):
    _plain_append_to(s, s["k"], s["ks"], s["new_k"])
    _plain_append_to(s, s["v"], s["vs"], s["new_v"])
    return _cache_of(s)


def _copy_pages(s, src, dst):
    for t in (_bytes(s["k"]), _bytes(s["v"]), s["ks"], s["vs"]):
        t[:, dst] = t[:, src]


def _plain_copy(s):
    _copy_pages(s, s["src"].long(), s["dst"].long())
    s["done"][:s["src"].numel()] = 1
    return _pages_answer(s)


def _plain_compact(s):
    table, refs = s["before"]
    used = refs > 0
    live = used.sum()
    index = torch.arange(refs.numel(), device="cuda")
    src, dst = torch.nonzero(used & (index >= live))[:, 0], torch.nonzero(~used & (index < live))[:, 0]
    to = torch.where(used, index, -1)
    to[src] = dst
    _copy_pages(s, src, dst)
    s["table"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    s["refs"].copy_(refs)
    s["refs"][dst] = refs[src]
    s["refs"][src] = 0
    s["live"][0] = live
    s["moved_to"].copy_(to)
    return _pages_answer(s)


def _plain_branch(s):
    ps, table, refs, held = s["case"]["page_size"], s["table"], s["refs"], s["held"]
    src, dst, lens, grown = (s[k].long() for k in ("src", "dst", "lens", "grown"))
    n, width = src.numel(), table.shape[1]
    # the old branches go
    gone = table[dst]
    refs.index_add_(0, gone.clamp(min=0).long().view(-1), -(gone >= 0).int().view(-1))
    table[dst] = -1
    # full pages are shared, the last one is copied where it is not full
    full, part = lens // ps, (lens % ps > 0).long()
    cols = torch.arange(width, device="cuda")
    shared = torch.where(cols < full[:, None], table[src], -1)
    refs.index_add_(0, shared.clamp(min=0).long().view(-1), (shared >= 0).int().view(-1))
    free = torch.sort((refs > 0).int(), stable=True)[1]  # pages in use last, else by number
    rank = part.cumsum(0)
    room = refs.numel() - (refs > 0).sum()
    new = free[(rank - 1).clamp(min=0)]
    old = table[src, full.clamp(max=width - 1)].long()
    table[dst] = torch.where((cols == full[:, None]) & (part > 0)[:, None], new[:, None].int(), shared)
    refs.index_add_(0, new, part.int())
    copied = torch.nonzero(part)[:, 0]
    _copy_pages(s, old[copied], new[copied])
    held[dst] = (full + part).int()
    s["done"][:n] = (rank <= room).int()
    # pages for the tokens to come
    want = (grown + ps - 1) // ps - held[dst].long()
    more = want.clamp(min=0)
    free = torch.sort((refs > 0).int(), stable=True)[1]
    room = refs.numel() - (refs > 0).sum()
    ends = more.cumsum(0)
    nth = cols - held[dst].long()[:, None]
    added = (nth >= 0) & (nth < more[:, None])
    pages = free[torch.where(added, (ends - more)[:, None] + nth, 0)]
    table[dst] = torch.where(added, pages.int(), table[dst])
    refs.index_add_(0, pages.view(-1), added.int().view(-1))
    held[dst] += more.int()
    s["roomy"][:n] = (ends <= room).int()
    return _pages_answer(s)


_PLAIN_PAGES = {"branch": _plain_branch, "compact": _plain_compact, "copy": _plain_copy}


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return _exact_append(s)
    return None  # whole numbers and copies


def _exact_sequence(case, codes, scales, pages, length):
    """[kv_heads, length, head_dim]: one sequence, page by page."""
    parts = []
    for p in pages:
        c = codes[0, p].to(torch.float64)
        parts.append(c * scales[0, p].double().repeat_interleave(case["scale_block"], -1)[..., None])
    return torch.cat(parts, 1)[:, :length]


def _exact_attend(s):
    case = s["case"]
    out, d, g = s["out"].double(), case["head_dim"], case["group"]
    lens, at, table = s["lens"].tolist(), s["offsets"].tolist(), s["table"].tolist()
    for b, length in enumerate(lens):
        n = at[b + 1] - at[b]
        if not n:
            continue
        if not length:
            out[at[b]:at[b + 1]] = 0
            continue
        pages = table[b][:-(-length // case["page_size"])]
        k, v = (_exact_sequence(case, s[c], s[c + "s"], pages, length) for c in "kv")
        q = s["q"][at[b]:at[b + 1]].double().view(n, -1, g, d)
        seen = torch.arange(length, device="cuda")[None, :] <= (torch.arange(n, device="cuda") + length - n)[:, None]
        if not case["causal"]:
            seen[:] = True
        for h in range(case["kv_heads"]):
            x = torch.einsum("ngd,kd->ngk", q[:, h], k[h]) / math.sqrt(d)
            x = x.masked_fill(~seen[:, None], -math.inf)
            most = x.amax(-1, keepdim=True)
            e = torch.exp(x - most.masked_fill(most.isinf(), 0.0))
            w = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            y = torch.einsum("ngk,kd->ngd", w, v[h])
            out[at[b]:at[b + 1], h * g * d:(h + 1) * g * d] = y.reshape(n, g * d)
    return out


def _exact_append(s):
    """By sequence and block.  A scale is the largest magnitude over the largest code, held in 32 bits, like its reciprocal and each
    quotient, since the codes hang on them."""
    case = s["case"]
    ps, sb, kind = case["page_size"], case["scale_block"], s["k"].dtype
    top = QMAX[case["type"]]
    held = lambda x: x.float().double()  # noqa: E731
    step = float(torch.tensor(1.0 / top, dtype=torch.float32))
    many, first, table, at = s["many"].tolist(), s["first"].tolist(), s["table"].tolist(), s["offsets"].tolist()

    def code(y):
        y = held(y)
        if kind == torch.int8:
            return torch.floor(y).add(((y - torch.floor(y) > 0.5) | ((y - torch.floor(y) == 0.5) & (torch.floor(y) % 2 == 1))).double()).clamp(-top, top)
        # e4m3: 3 bits behind the leading one, steps of 2^-9 at least
        unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return (torch.round(y / unit) * unit).clamp(-top, top)

    def one(codes, scales, new):
        c, sc = codes.to(torch.float64), scales.double()
        for b, n in enumerate(many):
            p0 = first[b]
            for lo in range(p0 // sb * sb, p0 + n, sb) if n else ():
                a, z = max(lo, p0), min(lo + sb, p0 + n)
                page, inside = table[b][lo // ps], lo % ps
                x = new[at[b] + a - p0:at[b] + z - p0].double().transpose(0, 1)  # head, token, dim
                before = sc[0, page, :, inside // sb].clone()
                now = held(x.abs().amax((1, 2)) * step)
                if a > lo:
                    now = torch.maximum(now, before)
                back = torch.where(now > 0, held(1 / now), torch.zeros_like(now))
                if a > lo:
                    old = c[0, page, :, inside:inside + a - lo]
                    c[0, page, :, inside:inside + a - lo] = code(old * held(before * back)[:, None, None])
                c[0, page, :, inside + a - lo:inside + z - lo] = code(x * back[:, None, None])
                sc[0, page, :, inside // sb] = now
        return c, sc

    if sum(many) * case["kv_heads"] > 8 * 512 * 96:
        return None
    k, ks = one(s["k"], s["ks"], s["new_k"])
    v, vs = one(s["v"], s["vs"], s["new_v"])
    codes = (k, v) if kind != torch.int8 else (None, None)  # whole numbers need none
    return {"k": codes[0], "v": codes[1], "k_scales": ks, "v_scales": vs}
