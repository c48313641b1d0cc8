"""A paged 8-bit key/value cache in plain torch on the CPU: what the liger_kv8_* operators are compared with."""
import ctypes as C

import numpy as np
import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def encode(x, kind):
    """fp32 -> code, to nearest even, saturated."""
    if kind == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def raw(t):
    return t.view(torch.uint8)


class Cache:
    """The arrays of a liger_kv8_cache on the CPU and, after to_gpu(), on the GPU with the C struct that names them."""

    def __init__(self, kind="int8", layers=1, num_pages=16, kv_heads=2, page_size=16, scale_block=16, head_dim=64, slots=4,
                 max_pages=8, seed=0, garbage=True):
        self.kind, self.layers, self.num_pages, self.kv_heads = kind, layers, num_pages, kv_heads
        self.page_size, self.scale_block, self.head_dim, self.slots, self.max_pages = page_size, scale_block, head_dim, slots, max_pages
        gen = torch.Generator().manual_seed(seed)
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        # what nobody wrote is anything: any byte (e4m3 NaN among them), any scale
        fill = lambda: torch.randint(0, 256, shape, dtype=torch.uint8, generator=gen) if garbage else torch.zeros(shape, dtype=torch.uint8)  # noqa: E731
        self.k, self.v = fill(), fill()
        blocks = (layers, num_pages, kv_heads, page_size // scale_block)
        self.ks, self.vs = (torch.full(blocks, float("nan") if garbage else 0.0) for _ in range(2))
        self.table = torch.full((slots, max_pages), -1, dtype=torch.int32)
        self.count = torch.zeros(slots, dtype=torch.int32)
        self.refs = torch.zeros(num_pages, dtype=torch.int32)
        self.gen = gen

    # ---- filling -----------------------------------------------------------------------------------------------------------
    def give_pages(self, lens):
        """Pages anywhere in the pool for slots 0 .. len(lens) - 1."""
        order = torch.randperm(self.num_pages, generator=self.gen).tolist()
        for slot, length in enumerate(lens):
            need = -(-length // self.page_size)
            for j in range(need):
                page = order.pop()
                self.table[slot, j] = page
                self.refs[page] += 1
            self.count[slot] = need

    def write(self, layer, slot, k, v):
        """Quantises [tokens, kv_heads, head_dim] fp32 values as the slot's first tokens, block by block."""
        for codes, scales, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
            for lo in range(0, x.shape[0], self.scale_block):
                part = x[lo:lo + self.scale_block]
                page, inside = int(self.table[slot, lo // self.page_size]), lo % self.page_size
                s = part.abs().amax((0, 2)) * torch.tensor(1.0 / QMAX[self.kind])
                back = torch.where(s > 0, 1.0 / s, 0.0)
                scales[layer, page, :, inside // self.scale_block] = s
                codes[layer, page, :, inside:inside + part.shape[0]] = raw(encode(part * back[None, :, None], self.kind)).transpose(0, 1)

    def fill(self, lens, layer=0, spread=1.0):
        """Random tokens for slots 0 ..; `spread` > 1 makes the blocks' scales differ by up to that."""
        for slot, n in enumerate(lens):
            if not n:
                continue
            k, v = (torch.randn((n, self.kv_heads, self.head_dim), generator=self.gen) for _ in range(2))
            if spread > 1.0:
                blocks = -(-n // self.scale_block)
                f = torch.exp2(torch.rand((blocks, self.kv_heads), generator=self.gen) * float(np.log2(spread)))
                v = v * f.repeat_interleave(self.scale_block, 0)[:n, :, None]
            self.write(layer, slot, k, v)

    def values(self, layer, slot, length):
        """[length, kv_heads, head_dim] in 64 bits: keys, values."""
        out = []
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            parts = []
            for j in range(-(-length // self.page_size)):
                page = int(self.table[slot, j])
                c = codes[layer, page].view(DTYPE[self.kind]).double()
                parts.append((c * scales[layer, page].double().repeat_interleave(self.scale_block, -1)[..., None]).transpose(0, 1))
            out.append(torch.cat(parts)[:length] if parts else torch.zeros((0, self.kv_heads, self.head_dim), dtype=torch.float64))
        return out

    # ---- the GPU's copy ----------------------------------------------------------------------------------------------------
    NAMES = ("k", "v", "ks", "vs", "table", "count", "refs")

    def to_gpu(self, liger):
        self.dev = {n: getattr(self, n).cuda() for n in self.NAMES}
        self.c = self.struct(liger, {n: t.data_ptr() for n, t in self.dev.items()})
        return self

    def struct(self, liger, at):
        c = liger.Kv8Cache()
        c.k_pages, c.v_pages, c.k_scales, c.v_scales = at["k"], at["v"], at["ks"], at["vs"]
        c.page_table, c.page_count, c.page_refs = at["table"], at["count"], at["refs"]
        c.layers, c.num_pages, c.kv_heads, c.page_size = self.layers, self.num_pages, self.kv_heads, self.page_size
        c.scale_block, c.head_dim, c.type = self.scale_block, self.head_dim, {"int8": 0, "e4m3": 1}[self.kind]
        c.slots, c.max_pages = self.slots, self.max_pages
        return c

    @property
    def by(self):
        return C.byref(self.c)

    def from_gpu(self):
        return {n: t.cpu() for n, t in self.dev.items()}


def attention(cache, layer, q, n, length, slot, scale, causal):
    """One sequence in 64 bits: q [n, heads, D] -> out [n, heads, D], and what its error bound is made of: sum p |v|, the
    largest sum |q k| scale log2(e) of a score, the largest |v|."""
    heads, d = q.shape[1], q.shape[2]
    if not n or not length:
        return torch.zeros((n, heads, d), dtype=torch.float64), torch.zeros((n, heads, d), dtype=torch.float64), 0.0, 0.0
    k, v = cache.values(layer, slot, length)
    g = heads // cache.kv_heads
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    q = q.double()
    x = torch.einsum("nhd,khd->hnk", q, k) * scale
    if causal:
        seen = torch.arange(length)[None, :] <= (torch.arange(n) + length - n)[:, None]
        x = x.masked_fill(~seen, -float("inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -float("inf"), 0.0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    size = float(torch.einsum("nhd,khd->hnk", q.abs(), k.abs()).max()) * abs(scale) * 1.4427
    return torch.einsum("hnk,khd->nhd", p, v), torch.einsum("hnk,khd->nhd", p, v.abs()), size, float(v.abs().max())


def attention_tolerance(want, mixed, size, d, weights16=None):
    """fp16 result: half a step, 2^-11 relative, or 2^-25 below the normal numbers.  A score is a sum of d products in fp32
    and is off by at most d * 2^-23 * sum |q k| (each of d additions rounds or truncates); in log2 units that is a relative error
    of ln 2 times it in a weight, once above and once below the fraction.  2^-18 * sum p |v| stands for the weights' other
    roundings: exp2 (2^-22), its argument (2^-24 times scores below 32), two fp16 parts (2^-22), the fp32 sums.
    weights16 = (keys, largest |v|): weights are rounded to one fp16 number each, 2^-11 relative, or 2^-25 below 2^-14, in units in
    which the largest weight's share of the sum is 1 and the largest value scale so far is the unit of v."""
    tol = want.abs() * 2.0 ** -11 + 2.0 ** -25 + mixed * (2 * 0.6932 * d * 2.0 ** -23 * size + 2.0 ** -18)
    return tol if weights16 is None else tol + mixed * 2.0 ** -11 + weights16[0] * weights16[1] * 2.0 ** -25


def append(cache, layer, slot, first, k, v):
    """The definition of liger_kv8_append for one sequence: k, v [n, kv_heads, D] fp16, changes the CPU arrays."""
    n, sb, ps, kind = k.shape[0], cache.scale_block, cache.page_size, cache.kind
    for codes, scales, x in ((cache.k, cache.ks, k), (cache.v, cache.vs, v)):
        for lo in range(first // sb * sb, first + n, sb) if n else ():
            a, z = max(lo, first), min(lo + sb, first + n)
            page, inside = int(cache.table[slot, lo // ps]), lo % ps
            new = x[a - first:z - first].float()
            s = new.abs().amax((0, 2)) * torch.tensor(1.0 / QMAX[kind])
            at = codes[layer, page].view(DTYPE[kind])
            if a > lo:
                old = scales[layer, page, :, inside // sb].clone()
                s = torch.maximum(s, old)
            fine = (s > 0) & s.isfinite()
            back = torch.where(fine, 1.0 / s, 0.0)
            if a > lo:
                ratio = torch.where(fine, old * back, 0.0)
                held = at[:, inside:inside + a - lo].float() * ratio[:, None, None]
                grown = (s != old)[:, None, None]
                again = encode(torch.where(fine[:, None, None], held, 0.0), kind).float()
                again = torch.where(grown, again, at[:, inside:inside + a - lo].float())
                raw(at)[:, inside:inside + a - lo] = raw(again.to(DTYPE[kind]))
            y = torch.where(fine[None, :, None], new * back[None, :, None], 0.0)
            raw(at)[:, inside + a - lo:inside + z - lo] = raw(encode(y, kind)).transpose(0, 1)
            scales[layer, page, :, inside // sb] = s


class Pages:
    """The page operators on plain lists."""

    def __init__(self, num_pages, slots, max_pages, page_size):
        self.n, self.slots, self.width, self.ps = num_pages, slots, max_pages, page_size
        self.table = [[] for _ in range(slots)]
        self.refs = [0] * num_pages

    def free_pages(self):
        return [p for p in range(self.n) if not self.refs[p]]

    def reserve(self, slots, lens):
        free, used, done, seen = self.free_pages(), 0, [], set()
        for slot, n in zip(slots, lens):
            ok = 0 <= slot < self.slots and n >= 0 and slot not in seen and -(-n // self.ps) <= self.width
            if 0 <= slot < self.slots:
                seen.add(slot)
            if ok:
                want = max(0, -(-n // self.ps) - len(self.table[slot]))
                pages = free[used:used + want]
                used += want
                ok = len(pages) == want
                if ok:
                    self.table[slot] += pages
                    for p in pages:
                        self.refs[p] = 1
            done.append(int(ok))
        return done

    def fork(self, src, dst, lens):
        """Also returns the pages that are copied, [(from, to)]."""
        free, used, done, seen, moves = self.free_pages(), 0, [], set(), []
        before = [list(r) for r in self.table]
        for s, d, n in zip(src, dst, lens):
            ok = 0 <= s < self.slots and 0 <= d < self.slots and n >= 0 and d not in seen
            if 0 <= d < self.slots:
                seen.add(d)
            ok = ok and s != d and not before[d] and -(-n // self.ps) <= len(before[s])
            if ok:
                full, part = n // self.ps, int(n % self.ps > 0)
                page = free[used:used + part]
                used += part
                ok = len(page) == part
                if ok:
                    for p in before[s][:full]:
                        self.refs[p] += 1
                    for p in page:
                        self.refs[p] = 1
                        moves.append((before[s][full], p))
                    self.table[d] = before[s][:full] + page
            done.append(int(ok))
        return done, moves

    def free(self, slots):
        for s in slots:
            if 0 <= s < self.slots:
                for p in self.table[s]:
                    self.refs[p] -= 1
                self.table[s] = []

    def copy(self, src, dst):
        owner = {}
        for i, d in enumerate(dst):
            if 0 <= d < self.n:
                owner.setdefault(d, i)
        done = [int(0 <= s < self.n and 0 <= d < self.n and owner[d] == i and (s == d or s not in owner)) for i, (s, d) in enumerate(zip(src, dst))]
        return done, [(s, d) for s, d, ok in zip(src, dst, done) if ok and s != d]

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if not self.refs[p]]
        late = [p for p in range(live, self.n) if self.refs[p]]
        to = [p if self.refs[p] else -1 for p in range(self.n)]
        for a, b in zip(late, holes):
            to[a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to[p] for p in row] for row in self.table]
        return live, to, list(zip(late, holes))

    def arrays(self):
        table = torch.full((self.slots, self.width), -1, dtype=torch.int32)
        for s, row in enumerate(self.table):
            table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        return table, torch.tensor([len(r) for r in self.table], dtype=torch.int32), torch.tensor(self.refs, dtype=torch.int32)
