"""The paged KV cache on the GPU: tables built from lengths, rows appended to
pages, attention of a batch behind a shared prefix, and the three in turn.

Whole numbers are compared for equality with a plain loop. Attention is
compared with the definition in 64 bits (`Attention`, which also says how far
a result may be off, from the roundings that the kernel makes).
"""
import ctypes
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
H, I32 = torch.float16, torch.int32
NAN, INF = float("nan"), float("inf")


def up(n, page):
    return -(-n // page)


def ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


# ------------------------------------------------------------------- tables --

def plain_tables(cached, added, free, table, page, rows):
    """The definition: (table, row_starts, lengths, slots, needed)."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    starts, lengths, slots, taken = [0], [], [-1] * rows, 0
    for b, (c, a) in enumerate(zip(cached, added)):
        c, a = max(c, 0), max(a, 0)
        for column in range(min(up(c, page), width),
                            min(up(c + a, page), width)):
            table[b][column] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(a):
            row, at = starts[b] + i, c + i
            if row >= rows:
                break
            if at // page < width and table[b][at // page] >= 0:
                slot = table[b][at // page] * page + at % page
                slots[row] = slot if slot < 2 ** 31 else -1
        starts.append(starts[b] + a)
        lengths.append(c + a)
    top = 2 ** 31 - 1
    return (table, [min(s, top) for s in starts],
            [min(n, top) for n in lengths], slots, [min(taken, top)])


def check_tables(pkg, cached, added, free, table, page, rows, pitch=0):
    width = len(table[0]) if table else 0
    buf = torch.full((len(table), width + pitch), 77, dtype=I32,
                     device="cuda")
    got = buf[:, :width]
    if width:
        got.copy_(ints(table))
    starts, lengths, slots, needed = pkg.page_tables(
        ints(cached), ints(added), ints(free), got, page, rows)
    want = plain_tables(cached, added, free, table, page, rows)
    for g, w, n in zip((got, starts, lengths, slots, needed), want,
                       ("table", "starts", "lengths", "slots", "needed")):
        assert g.dtype == I32 and g.tolist() == w, n
    assert bool((buf[:, width:] == 77).all()), "write past the table's rows"


@pytest.mark.parametrize("batch", [0, 1, 2, 63, 64, 65, 511, 512, 513, 1500])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_tables(pkg, dev, batch, page):
    g = torch.Generator().manual_seed(batch * 100 + page)

    def draw(lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=g).tolist()

    print(f"tables {batch} {page}", flush=True)
    cached, added = draw(0, 60, batch), draw(0, 30, batch)
    width = up(90, page) + 2
    free = torch.randperm(40 * batch + 99, generator=g).tolist()
    table = [[draw(0, 5000, 1)[0] if c < up(n, page) else -9
              for c in range(width)] for n in cached]
    total = sum(added)
    need = sum(up(c + a, page) - up(c, page) for c, a in zip(cached, added))
    for rows, have, pitch in ((total, need, 0), (total + 40, need + 9, 3),
                              (total // 2, need // 2, 0), (0, 0, 1)):
        check_tables(pkg, cached, added, (free * 30)[:have], table, page,
                     rows, pitch)


def test_tables_one_long_request(pkg, dev):
    """Many rows of one request among single tokens; no tokens at all."""
    added = [1] * 40 + [9000] + [0] * 5 + [1] * 30
    cached = [17 * i % 50 for i in range(len(added))]
    table = [[3 * i + c for c in range(600)] for i in range(len(added))]
    check_tables(pkg, cached, added, list(range(2000)), table, 16,
                 sum(added))
    check_tables(pkg, cached, [0] * len(added), [5], table, 16, 12)


def test_tables_bounds(pkg, dev):
    """Requests longer than their table's row, counts below 0 and at the type's
    end, pages whose slots pass 32 bits, rows without a table."""
    top = 2 ** 31 - 1
    table = [[1, 2, 3]] * 6
    check_tables(pkg, [0, 40, 47, 48, 200, -5], [70, 9, 1, 3, 4, 20],
                 list(range(9)), table, 16, 107)
    # 600 such requests: sums past 32 bits, in more than one round
    check_tables(pkg, [top, -top - 1, 5] * 200, [top, -3, top] * 200,
                 list(range(7)), [[4, 4]] * 600, 16, 50)
    check_tables(pkg, [15, 0], [1, 2], [top, 2 ** 27], [[2 ** 27], [-1]],
                 16, 3)
    check_tables(pkg, [15, 0], [1, 2], [2 ** 27 - 1], [[2 ** 27 - 1], [-1]],
                 16, 3)
    check_tables(pkg, [3, 0], [1, 2], [], [[], []], 16, 3)
    check_tables(pkg, [0], [top], [], [[0, 0]], top, 2)


# ------------------------------------------------------------------- append --

def plain_append(cache, rows, slots):
    flat = cache.transpose(1, 2).reshape(-1, *cache.shape[1::2]).clone()
    for r, s in enumerate(slots):
        if 0 <= s < flat.shape[0]:
            flat[s] = rows[r]
    return flat.unflatten(0, cache.shape[::2][:2]).transpose(1, 2)


def new_cache(g, pages, heads, page, d, token_major=False, pad=0):
    """A cache and the buffer it is a view of."""
    shape = (pages, page, heads) if token_major else (pages, heads, page)
    buf = torch.randn(*shape, d + pad, generator=g).half().cuda()
    view = buf[..., :d]
    return (view.permute(0, 2, 1, 3) if token_major else view), buf


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("rows,heads,d,dv,page,pages", [
    (1, 1, 8, 8, 1, 1), (5, 3, 64, 64, 16, 4), (70, 8, 128, 128, 16, 9),
    (333, 2, 40, 24, 7, 60), (9, 32, 256, 200, 24, 3),
    (5000, 2, 64, 128, 64, 90)])
def test_append(pkg, dev, token_major, rows, heads, d, dv, page, pages):
    g = torch.Generator().manual_seed(rows + d)
    print(f"append {rows} {heads} {d} {dv} {page}", flush=True)
    kc, kbuf = new_cache(g, pages, heads, page, d, token_major, pad=8)
    vc, vbuf = new_cache(g, pages, heads, page, dv, token_major)
    # rows of one fused buffer, heads apart by more than their size
    kv = torch.randn(rows, heads, d + dv + 16, generator=g).half().cuda()
    k, v = kv[..., :d], kv[..., d + 8:d + 8 + dv]
    slots = torch.randperm(pages * page, generator=g)[:rows].tolist()
    slots += [-1] * (rows - len(slots))
    if rows > 3:  # outside the cache
        slots[1], slots[2], slots[3] = -1, pages * page, -2 ** 31
        slots[0] = 2 ** 31 - 1 if rows > 5 else slots[0]
    want_k = plain_append(kc, k, slots)
    want_v = plain_append(vc, v, slots)
    beside = kbuf[..., d:].clone()
    pkg.append_kv(k, v, kc, vc, ints(slots))
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    assert torch.equal(kbuf[..., d:], beside)


def test_append_far_pages(pkg, dev):
    """Pages whose elements pass 32 bits."""
    pages, heads, page, d = 5, 1, 2, 8
    stride = 1 << 30  # elements: 4 pages reach 2^32
    buf = torch.zeros(stride * (pages - 1) + 64, dtype=H, device="cuda")
    kc = buf.as_strided((pages, heads, page, d), (stride, 16, 8, 1))
    vc = torch.zeros(pages, heads, page, d, dtype=H, device="cuda")
    k = torch.arange(1, 17, device="cuda").half().reshape(2, 1, 8)
    pkg.append_kv(k, k, kc, vc, ints([9, 7]))
    assert torch.equal(kc[4, 0, 1], k[0, 0]) and torch.equal(kc[3, 0, 1],
                                                             k[1, 0])
    assert int((kc != 0).sum()) == 16 and int((buf[:4096] != 0).sum()) == 0
    q = torch.ones(1, 1, 8, dtype=H, device="cuda")
    o = pkg.shared_prefix_attention(q, kc, kc, ints([0, 1]), ints([1]),
                                    ints([[4]]), ints([3]), 2)
    # keys: place 0 and 1 of page 3 (0 and k[1]), place 0 of page 4 (0)
    w = torch.softmax(torch.tensor([0.0, float(k[1].sum()) * 8 ** -0.5, 0.0],
                                   dtype=torch.float64), 0)[1]
    assert (o[0, 0].double().cpu() - w * k[1, 0].double().cpu()).abs().max() \
        <= 16 * 2 ** -11 * 2


# ---------------------------------------------------------------- attention --

class Attention:
    """A batch's tensors, their definition in 64 bits, and how far a result
    may be off it.

    The kernel rounds each weight 2^(s - m) <= 1 to f16, by 2^-11 of it or, under
    2^-14, by 2^-25, sums the rounded ones, and rounds the result. Over a row's
    n keys the sum is at least 1 (the largest weight is 1), so with p the
    softmax and A = sum p |v| + |o|
      |got - o| <= 2^-11 |o| + 2^-11 A + n 2^-25 (max |v| + |o|) + 2^-25
    (the last: a result in f16's subnormal range), to which the 32-bit sums
    add n 2^-24 A and the scores (d + 8) 2^-24 S A, S = max_j scale sum |q k_j|
    (the scale's and the logarithm's roundings among the 8), all to first
    order: 2 % more, for exp2's last bit and the products of these.
    """

    def __init__(self, cached, added, heads, hk, d, dv, page, prefix=0, pad=0,
                 spare=1, token_major=False, seed=0, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.cached, self.added, self.prefix = cached, added, prefix
        self.heads, self.hk, self.d, self.dv, self.page = heads, hk, d, dv, page
        self.rows = sum(added) + pad
        lengths = [c + a for c, a in zip(cached, added)]
        lead = up(prefix, page)
        held = [up(n, page) for n in lengths]
        pages = lead + sum(held) + 2
        order = torch.randperm(pages, generator=g).tolist()
        self.prefix_pages = order[:lead]
        width = max(held + [0]) + spare
        self.table, at = [], lead
        for n in held:
            self.table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.width, self.lengths = width, lengths
        self.starts = [sum(added[:b]) for b in range(len(added) + 1)]
        self.q = (torch.randn(self.rows, heads, d, generator=g)
                  * q_scale).half().cuda()
        self.kc, _ = new_cache(g, pages, hk, page, d, token_major)
        self.vc, _ = new_cache(g, pages, hk, page, dv, token_major)
        # tokens past the lengths, and the pages of no one, hold anything
        taken = torch.zeros(pages, page, dtype=torch.bool)
        for pp, n in [(self.prefix_pages, prefix)] + list(
                zip(self.table, lengths)):
            for j in range(n):
                taken[pp[j // page], j % page] = True
        rest = (~taken).cuda()
        for c in (self.kc, self.vc):
            c.transpose(1, 2)[rest] = NAN
        self.scale = d ** -0.5

    def call(self, pkg, o=None, **kw):
        if o is None:
            o = torch.full((self.rows, self.heads, self.dv), 9.0, dtype=H,
                           device="cuda")
        batch = len(self.added)
        table = (ints(self.table) if batch and self.width else
                 torch.empty(batch, self.width, dtype=I32, device="cuda"))
        out = pkg.shared_prefix_attention(
            self.q, self.kc, self.vc, ints(self.starts), ints(self.lengths),
            table, ints(self.prefix_pages), self.prefix, o, **kw)
        assert out is o
        return o

    def keys(self, b, g):
        """(K, V) of request b's prefix and own tokens, in 64 bits; a page
        that is not in the cache is zeros that `there` tells."""
        ks, vs, there = [], [], []
        for pages, n in ((self.prefix_pages, self.prefix),
                         (self.table[b], self.lengths[b])):
            n = max(0, min(n, len(pages) * self.page))
            for j in range(n):
                p = pages[j // self.page]
                ok = 0 <= p < self.kc.shape[0]
                there.append(ok)
                ks.append(self.kcpu[p, g, j % self.page] if ok else
                          torch.zeros(self.d, dtype=torch.float64))
                vs.append(self.vcpu[p, g, j % self.page] if ok else
                          torch.zeros(self.dv, dtype=torch.float64))
        if not ks:
            return (torch.zeros(0, self.d, dtype=torch.float64),
                    torch.zeros(0, self.dv, dtype=torch.float64),
                    torch.zeros(0, dtype=torch.bool))
        return torch.stack(ks), torch.stack(vs), torch.tensor(there)

    def expected(self):
        """(o, bound), NaN where the rows are not written."""
        self.kcpu, self.vcpu = self.kc.double().cpu(), self.vc.double().cpu()
        q = self.q.double().cpu()
        o = torch.full((self.rows, self.heads, self.dv), NAN,
                       dtype=torch.float64)
        bound = o.clone()
        group = self.heads // self.hk
        for b, a in enumerate(self.added):
            first = self.starts[b]
            if not a:
                continue
            for g in range(self.hk):
                k, v, there = self.keys(b, g)
                own = torch.arange(len(k)) - self.prefix
                for i in range(a):
                    sees = there & ((own < 0)
                                    | (own <= self.lengths[b] - a + i))
                    kk, vv = k[sees], v[sees]
                    for h in range(g * group, (g + 1) * group):
                        row = q[first + i, h]
                        if not len(kk):
                            o[first + i, h] = bound[first + i, h] = 0
                            continue
                        s = kk @ row * self.scale
                        p = torch.softmax(s, 0)
                        r = p @ vv
                        big = (kk.abs() @ row.abs()).max() * abs(self.scale)
                        spread = p @ vv.abs() + r.abs()
                        n = len(kk)
                        far = (2 ** -11 * (r.abs() + spread) + 2 ** -25
                               + n * 2 ** -25 * (vv.abs().amax(0) + r.abs())
                               + (n + (self.d + 8) * big) * 2 ** -24 * spread)
                        o[first + i, h] = r
                        bound[first + i, h] = 1.02 * far
        return o, bound

    def check(self, got):
        want, bound = self.expected()
        got = got.double().cpu()
        written = ~want.isnan()
        assert bool((got[~written] == 9).all()), "a row past the last"
        off = (got - want).abs()[written] - bound[written]
        assert bool((off <= 0).all()), float(off.max())
        return want


# tokens, drafts and prompts; few keys and many; sizes short of their bucket
SHAPES = [
    # cached, added, heads, kv heads, d, dv, page, prefix
    ([5], [1], 1, 1, 8, 8, 16, 0),
    ([0], [1], 4, 4, 64, 64, 16, 0),
    ([0], [1], 8, 1, 128, 128, 16, 1),
    ([3, 0, 40, 31], [1, 1, 1, 1], 9, 3, 64, 64, 16, 64),
    ([100, 7, 0, 333], [1, 1, 1, 1], 8, 2, 128, 128, 7, 300),
    ([0, 9, 60], [3, 0, 5], 6, 2, 80, 80, 24, 33),
    ([10, 0, 200], [2, 17, 1], 4, 1, 192, 128, 8, 100),
    ([63, 64, 65], [1, 2, 4], 2, 2, 256, 256, 64, 31),
    ([0, 50], [40, 33], 6, 2, 96, 96, 16, 0),
    ([20, 0, 5], [70, 130, 2], 8, 2, 64, 64, 32, 96),
    ([12], [150], 3, 1, 128, 128, 16, 129),
    ([0, 1], [64, 64], 2, 1, 40, 24, 5, 65),
    ([1000], [1], 8, 1, 64, 64, 16, 2000),
    ([700, 3, 0], [1, 1, 1], 4, 2, 128, 128, 1, 40),
    # small requests around ones of more than 16 rows, behind a prefix
    ([30, 5, 200, 9], [1, 60, 2, 1], 8, 2, 96, 96, 16, 150),
    ([0, 3, 40, 0, 7, 90, 1], [40, 1, 0, 33, 1, 16, 17], 4, 4, 80, 64, 24, 70),
    ([5, 600, 0, 2], [1, 1, 20, 1], 24, 3, 192, 128, 32, 513),
]


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(pkg, dev, shape, token_major):
    cached, added, heads, hk, d, dv, page, prefix = shape
    print(f"attention {shape} {token_major}", flush=True)
    a = Attention(cached, added, heads, hk, d, dv, page, prefix, pad=3,
                  token_major=token_major, seed=len(cached) + d)
    a.check(a.call(pkg))


@pytest.mark.parametrize("batch", [33, 64, 65, 200])
def test_attention_batches(pkg, dev, batch):
    """Requests are found among their tiles, 64 at a step."""
    g = torch.Generator().manual_seed(batch)
    cached = torch.randint(0, 70, (batch,), generator=g).tolist()
    added = torch.randint(0, 4, (batch,), generator=g).tolist()
    print(f"batch {batch}", flush=True)
    for prefix in (0, 50):
        a = Attention(cached, added, 2, 1, 64, 64, 16, prefix, seed=batch)
        a.check(a.call(pkg))
    # a table wide enough for parts, and every tenth request of 30 rows or so
    added[::10] = [n + 14 for n in added[::10]]
    a = Attention(cached, added, 2, 1, 64, 64, 16, 130, seed=batch, spare=40)
    a.check(a.call(pkg))


def test_attention_empty(pkg, dev):
    """Requests without keys or rows, a batch of them, no rows at all."""
    a = Attention([0, 0], [0, 0], 2, 1, 64, 64, 16, 40, pad=4)
    a.check(a.call(pkg))
    # fewer tokens than new rows: the first rows see only the prefix, or none
    for prefix in (0, 40):
        a = Attention([0, 0, 9], [3, 40, 2], 4, 2, 64, 64, 16, prefix)
        a.lengths = [1, 7, 0]
        want = a.check(a.call(pkg))
        assert bool((want[:2] == 0).all()) == (prefix == 0)
        # a length below 0 is none
        a.lengths = [-4, 7, -2 ** 31]
        o = a.call(pkg)
        a.lengths = [0, 7, 0]
        a.check(o)
    # a table without columns, a cache without pages
    a = Attention([0], [2], 2, 1, 64, 64, 16, 20, spare=0)
    a.table, a.width = [[]], 0
    a.check(a.call(pkg))
    a.kc, a.vc = a.kc[:0], a.vc[:0]
    assert bool((a.call(pkg) == 0).all())
    a = Attention([], [], 2, 1, 64, 64, 16, 20, pad=2)
    assert bool((a.call(pkg) == 9).all())


@pytest.mark.parametrize("added", [[1, 1, 1], [60, 2, 33]])
def test_attention_pages_outside_the_cache(pkg, dev, added):
    """Tokens in pages that the cache does not have are not seen; lengths past
    the table's row stop there."""
    a = Attention([40, 100, 70], added, 4, 2, 64, 64, 16, 70, spare=0)
    pages = a.kc.shape[0]
    a.table[0][1], a.table[1][0] = -1, pages
    a.table[2][2] = 2 ** 31 - 1
    a.prefix_pages[1] = -2 ** 31
    a.check(a.call(pkg))
    a.prefix_pages = [pages + 5] * len(a.prefix_pages)
    a.table = [[-1] * a.width] * 3
    assert bool((a.call(pkg) == 0).all())
    a = Attention([40, 100, 70], added, 4, 2, 64, 64, 16, 0, spare=0)
    a.lengths = [n + 1000 for n in a.lengths]
    full = a.width * 16
    a.table[0] = a.table[1] = a.table[2] = max(a.table, key=lambda t: min(t))
    a.vc.nan_to_num_(0.5)
    a.kc.nan_to_num_(0.5)
    o = a.call(pkg)
    assert a.lengths[0] > full
    a.check(o)


def test_attention_infinities(pkg, dev):
    """A NaN in a row's query, or in a key that it sees, makes it NaN and no
    other request's; keys it does not see do nothing to it."""
    a = Attention([40, 9, 300], [1, 2, 1], 4, 2, 64, 64, 16, 70)
    want = a.call(pkg).clone()
    a.q[1, 2, 5] = NAN
    o = a.call(pkg)
    bad = o.isnan().all(-1)
    assert bool(bad[1, 2]) and int(o.isnan().any(-1).sum()) == 1
    assert torch.equal(o[~bad], want[~bad])
    a.q[1, 2, 5] = 0.5
    want = a.call(pkg).clone()
    # a key of request 2's own: its row alone
    p, at = a.table[2][100 // 16], 100 % 16
    a.kc[p, 1, at, 3] = NAN
    o = a.call(pkg)
    assert bool(o[3, 2:].isnan().all()) and not bool(o[3, :2].isnan().any())
    assert torch.equal(o[:3], want[:3])
    a.kc[p, 1, at, 3] = 0.5
    # an infinite value of the prefix reaches every row's column
    a.vc[a.prefix_pages[0], 0, 3, 7] = INF
    o = a.call(pkg)
    assert bool(o[:4, :2, 7].isinf().all())
    assert torch.equal(o[:4, 2:], a.call(pkg)[:4, 2:])
    assert bool(o[:4, 2:].isfinite().all())
    a.vc[a.prefix_pages[0], 0, 3, 7] = 0
    # scores far apart, at f16's largest values
    a.q.fill_(1.0)
    a.kc.nan_to_num_(0.0)
    a.kc.mul_(0.0)
    a.kc[a.prefix_pages[0], :, 0] = -65504.0
    a.kc[a.table[1][0], :, 0] = 65504.0
    a.vc.nan_to_num_(0.0)
    o = a.call(pkg)
    top = a.vc[a.table[1][0], :, 0].repeat_interleave(2, 0)
    assert torch.equal(o[1], top) and torch.equal(o[2], top)
    a.check(o)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_attention_scale(pkg, dev, scale):
    a = Attention([40, 9], [1, 50], 4, 2, 64, 64, 16, 70)
    a.scale = scale
    a.check(a.call(pkg, scale=scale))


def test_attention_strides(pkg, dev):
    """q and o as parts of wider rows, heads out of order in memory."""
    a = Attention([40, 9, 0], [1, 2, 20], 6, 2, 64, 64, 16, 70, pad=2)
    wide = torch.full((a.rows, 3 * 64 * 6 + 8), 7.0, dtype=H, device="cuda")
    q = wide[:, 64:64 + 64 * 6].unflatten(1, (6, 64))
    q.copy_(a.q)
    a.q = q
    o = wide[:, 64 * 7 + 4:64 * 13 + 4].unflatten(1, (6, 64))
    o.fill_(9.0)
    a.check(a.call(pkg, o))
    o.fill_(7.0)
    q.fill_(7.0)
    assert bool((wide == 7).all()), "write past o's rows"
    # [head, row] order
    buf = torch.full((6, a.rows, 64), 9.0, dtype=H, device="cuda")
    a.q = torch.randn(6, a.rows, 64, device="cuda").half().transpose(0, 1)
    a.check(a.call(pkg, buf.transpose(0, 1)))


def test_attention_workspaces(pkg, dev):
    """No workspace, short ones and all it can use give the same within the
    roundings; nothing past its end or in its first 256 KiB is written."""
    a = Attention([900, 40, 300], [1, 2, 1], 8, 2, 64, 64, 16, 1500)
    args = pkg.PagedAttentionArgs(
        q=a.q.data_ptr(), rows=a.rows, heads=8, batch=3, table_width=a.width,
        table_stride=a.width, prefix_length=a.prefix, scale=a.scale)
    keep = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
    for n, t in zip(("row_starts", "lengths", "block_table", "prefix_pages"),
                    keep):
        setattr(args, n, t.data_ptr())
    c = args.cache
    c.k, c.v = a.kc.data_ptr(), a.vc.data_ptr()
    c.pages, c.kv_heads, c.page_size, c.head_dim = a.kc.shape
    c.head_dim_v = 64
    c.k_strides[:], c.v_strides[:] = a.kc.stride()[:3], a.vc.stride()[:3]
    args.q_strides[:] = args.o_strides[:] = a.q.stride()[:2]
    lib, s = pkg.library(), torch.cuda.current_stream().cuda_stream
    full = lib.iree_mi355x_shared_prefix_attention_workspace_bytes(
        ctypes.byref(args))
    head = 256 << 10
    assert full > head
    for size in (0, 100, head, head + 5000, full - 1, full, full + 4096):
        ws = torch.full((size + 256,), 0xA5, dtype=torch.uint8,
                        device="cuda")
        o = torch.full((a.rows, 8, 64), 9.0, dtype=H, device="cuda")
        args.o = o.data_ptr()
        print(f"workspace {size} of {full}", flush=True)
        assert lib.iree_mi355x_shared_prefix_attention_f16(
            ctypes.byref(args), ws.data_ptr() if size else None, size,
            s) == pkg.OK
        a.check(o)
        assert bool((ws[size:] == 0xA5).all()) and bool(
            (ws[:min(size, head)] == 0xA5).all())


def test_two_streams_and_capture(pkg, dev):
    """Calls on two streams at once, and two graphs captured on one stream and
    replayed together, with eager calls between."""
    batches = [Attention([900, 40, 300 + s], [1, 2, 1], 8, 2, 64, 64, 16,
                         1500 + s, seed=s) for s in range(2)]
    want = [a.call(pkg).clone() for a in batches]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for a, s, g in zip(batches, streams, got):
            with torch.cuda.stream(s):
                g.append(a.call(pkg))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(o, w) for o in g)
    graphs, outs = [], []
    state = []
    for a in batches:
        t = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
        o = torch.empty_like(want[0])
        state.append(t)
        outs.append(o)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            pkg.shared_prefix_attention(a.q, a.kc, a.vc, *t, a.prefix, o)
        graphs.append(graph)
    for turn in range(4):
        for o in outs:
            o.fill_(3.0)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = batches[0].call(pkg)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), turn
        assert torch.equal(eager, want[0])
    # the captured call reads the lengths of its replay
    state[0][1].copy_(ints([500, 42, 301]))
    graphs[0].replay()
    batches[0].lengths = [500, 42, 301]
    torch.cuda.synchronize()
    batches[0].check(outs[0])


# Tables that could name more than 1024 keys, so that tiles are shared out and
# their parts joined, whatever the lengths are in the end.

def columns(page, keys=1100):
    return up(keys, page)


@pytest.mark.parametrize("shape", SHAPES)
def test_attention_parts(pkg, dev, shape):
    cached, added, heads, hk, d, dv, page, prefix = shape
    print(f"parts {shape}", flush=True)
    a = Attention(cached, added, heads, hk, d, dv, page, prefix, pad=3,
                  spare=columns(page), seed=len(cached) + d)
    a.check(a.call(pkg))


@pytest.mark.parametrize("spare", [0, 80])
@pytest.mark.parametrize("added", [[1, 1, 1, 1], [150, 1, 40, 3]])
@pytest.mark.parametrize("d, dv", [(192, 128), (160, 96), (136, 128),
                                   (128, 192), (200, 128)])
def test_attention_unequal_head_dims(pkg, dev, d, dv, added, spare):
    print(f"unequal {d} {dv} {added} {spare}", flush=True)
    a = Attention([70, 9, 0, 300], added, 6, 2, d, dv, 16, 100, pad=1,
                  spare=spare, seed=d)
    a.check(a.call(pkg))


@pytest.mark.parametrize("spare", [0, 80])
@pytest.mark.parametrize("heads, hk", [(200, 200), (600, 600), (130, 1),
                                       (260, 2), (17, 1)])
def test_attention_many_heads(pkg, dev, heads, hk, spare):
    """More KV heads than workgroups; a token's rows past a tile."""
    print(f"heads {heads} {hk} {spare}", flush=True)
    a = Attention([70, 0, 9], [1, 3, 2], heads, hk, 16, 16, 16, 40, pad=1,
                  spare=spare)
    a.check(a.call(pkg))


@pytest.mark.parametrize("prefix", [0, 30])
def test_attention_large_batch(pkg, dev, prefix):
    g = torch.Generator().manual_seed(prefix)
    cached = torch.randint(0, 30, (1500,), generator=g).tolist()
    added = torch.randint(0, 3, (1500,), generator=g).tolist()
    for spare in (0, columns(16)):
        print(f"large batch {prefix} {spare}", flush=True)
        a = Attention(cached, added, 1, 1, 8, 8, 16, prefix, pad=1,
                      spare=spare)
        a.check(a.call(pkg))


@pytest.mark.parametrize("first", [0, 40, 1008])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_padded_batch(pkg, dev, d, first):
    """A step padded to 1024 requests, of which 16 that follow one another have
    rows: they share the prefix as a batch of 16 does, to the last bit."""
    print(f"padded {d} {first}", flush=True)
    cached = [9, 0, 33, 70] * 4
    a = Attention(cached, [1, 2, 1, 3] * 4, 8, 2, d, d, 16, 3000, pad=1,
                  spare=columns(16), seed=d)
    want = a.call(pkg).clone()
    a.check(want)
    rest = 1024 - first - 16
    a.added = [0] * first + a.added + [0] * rest
    a.starts = [0] * first + a.starts + [a.starts[-1]] * rest
    a.lengths = [5] * first + a.lengths + [0] * rest
    a.table = ([a.table[0]] * first + a.table + [[-1] * a.width] * rest)
    assert torch.equal(a.call(pkg), want)


def test_attention_long_prefix_of_longer_keys(pkg, dev):
    """192-wide keys whose prefix has wide tiles though every request is
    small."""
    a = Attention([9, 0, 33, 70] * 6, [1, 2, 0, 3] * 6, 4, 1, 192, 128, 16,
                  1300, pad=1, seed=6)
    a.check(a.call(pkg))


@pytest.mark.parametrize("seed", range(12))
def test_attention_drawn(pkg, dev, seed):
    """Small and large requests in any order, lengths around a part's ends."""
    g = torch.Generator().manual_seed(seed)

    def one(*of):
        return of[int(torch.randint(0, len(of), (1,), generator=g))]

    batch = one(1, 2, 5, 9)
    cached = [one(0, 1, 63, 64, 65, 200, 321, 700) for _ in range(batch)]
    added = [one(0, 1, 1, 2, 5, 16, 17, 40, 130) for _ in range(batch)]
    hk = one(1, 2, 3)
    heads, d = hk * one(1, 3, 4, 8), one(8, 40, 64, 80, 128, 192)
    page, prefix = one(1, 5, 16, 64, 100), one(0, 0, 1, 64, 127, 450, 1300)
    print(f"drawn {cached} {added} {heads} {hk} {d} {page} {prefix}",
          flush=True)
    a = Attention(cached, added, heads, hk, d, min(d, 128), page, prefix,
                  pad=one(0, 1, 7), spare=one(0, 1, columns(page)),
                  token_major=one(False, True), seed=seed)
    a.check(a.call(pkg))


@pytest.mark.parametrize("batch", [33, 65, 200])
def test_attention_batches_parts(pkg, dev, batch):
    g = torch.Generator().manual_seed(batch + 1)
    cached = torch.randint(0, 70, (batch,), generator=g).tolist()
    added = torch.randint(0, 4, (batch,), generator=g).tolist()
    print(f"batch {batch}", flush=True)
    for prefix in (0, 50, 700):
        a = Attention(cached, added, 4, 2, 64, 64, 16, prefix, seed=batch,
                      spare=columns(16), pad=2)
        a.check(a.call(pkg))
        added[::10] = [n + 14 for n in added[::10]]


@pytest.mark.parametrize("added", [[1, 1, 1], [60, 2, 33], [0, 0, 0]])
def test_attention_pages_outside_the_cache_parts(pkg, dev, added):
    """Pages that the cache does not have, lengths below 0, requests without
    rows, where there are parts."""
    a = Attention([40, 1000, 70], added, 4, 2, 64, 64, 16, 1500, pad=1,
                  spare=columns(16))
    pages = a.kc.shape[0]
    a.table[0][1], a.table[1][0] = -1, pages
    a.table[1][30:50] = [2 ** 31 - 1] * 20
    a.prefix_pages[20:60] = [-2 ** 31] * 40
    a.check(a.call(pkg))
    a.prefix_pages = [pages + 5] * len(a.prefix_pages)
    a.table = [[-1] * a.width] * 3
    rows = sum(added)
    assert bool((a.call(pkg)[:rows] == 0).all())
    a.prefix, a.prefix_pages = 0, []
    a.lengths = [-1, -2 ** 31, 0]
    o = a.call(pkg)
    assert bool((o[:rows] == 0).all()) and bool((o[rows:] == 9).all())


def test_attention_row_starts(pkg, dev):
    """Starts below 0, past the rows or out of order: rows stay within the
    tensors, and requests in order get their rows."""
    a = Attention([40, 9, 30, 4], [2, 3, 20, 1], 4, 2, 64, 64, 16, 70, pad=3)
    for spare in (0, columns(16)):
        a.table = [r + [-1] * spare for r in a.table]
        a.width += spare
        a.starts = [0, 2, 5, 25, 26]
        a.check(a.call(pkg))
        want, bound = a.expected()
        # request 3's end lies past the rows: the padding is its. The others'
        # rows have their keys (the parts' ends move with all requests' rows,
        # so not the same roundings).
        a.starts[4] = 2 ** 31 - 1
        o = a.call(pkg)
        assert bool(((o.double().cpu() - want).abs() <= bound)[:25].all())
        assert not bool((o == 9).all(-1).any())
        for starts in ([-5, -1, 5, 25, 26], [7, 2, 25, 5, 26],
                       [-2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1, 3]):
            a.starts = starts
            a.call(pkg)
    torch.cuda.synchronize()


@pytest.mark.parametrize("added", [2, 40])
def test_attention_long_lines(pkg, dev, added):
    """A table that could name 2^26 keys a request: keys are shared out in
    larger units, with few and with many rows."""
    page, batch = 1 << 16, 40
    cached = [9000, 70, 3000] + [7 * i % 40 for i in range(batch - 3)]
    a = Attention(cached, [added, 1, 0, added] + [1] * (batch - 4), 2, 1, 8,
                  8, page, 100, spare=1023)
    a.check(a.call(pkg))


@pytest.mark.parametrize("added", [1, 40])
def test_attention_far_pages(pkg, dev, added):
    """Pages of a cache past 2^32 elements, for narrow and wide tiles."""
    a = Attention([20, 9], [added, 2], 2, 1, 8, 8, 16, 20, spare=columns(16))
    want = a.call(pkg).clone()
    pages = a.kc.shape[0]
    buf = torch.zeros((1 << 30) * (pages - 1) + 128, dtype=H, device="cuda")
    far = buf.as_strided(a.kc.shape, (1 << 30, 128, 8, 1))
    far.copy_(a.kc)
    a.kc = far
    assert torch.equal(a.call(pkg), want)
    a.check(want)


def test_stream_argument(pkg, dev):
    """Each call on the stream that it names, behind that stream's work."""
    a = Attention([900, 40], [1, 30], 4, 2, 64, 64, 16, 1500)
    want = a.call(pkg).clone()
    table, page = ints([[3, -1, -1], [5, 6, -1]]), 16
    k = torch.randn(4, 2, 64, device="cuda").half()
    caches = [torch.zeros(9, 2, page, 64, dtype=H, device="cuda")
              for _ in range(2)]
    free, cached, added = ints([1, 2, 7]), ints([15, 30]), ints([2, 2])
    o = torch.empty_like(want)
    lengths = torch.zeros(2, dtype=I32, device="cuda")
    t = [ints(a.starts), lengths, ints(a.table), ints(a.prefix_pages)]
    late = ints(a.lengths)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):  # the lengths arrive behind some work
        for _ in range(10):
            big = big @ big * 1e-3
        lengths.copy_(late)
    pkg.shared_prefix_attention(a.q, a.kc, a.vc, *t, a.prefix, o, stream=s)
    starts, total, slots, needed = pkg.page_tables(
        cached, added, free, table, page, 4, stream=s)
    pkg.append_kv(k, k, *caches, slots, stream=s)
    s.synchronize()
    assert torch.equal(o, want)
    assert table.tolist() == [[3, 1, -1], [5, 6, -1]]
    assert slots.tolist() == [3 * 16 + 15, 16, 6 * 16 + 14, 6 * 16 + 15]
    assert needed.tolist() == [1] and total.tolist() == [17, 32]
    for c in caches:
        flat = c.transpose(1, 2).reshape(-1, 2, 64)
        assert torch.equal(flat[slots.long()], k)


@pytest.mark.parametrize("raw", [False, True])
@pytest.mark.parametrize("operator", ["page_tables", "attention"])
def test_results_on_another_stream(pkg, dev, operator, raw):
    """The results of a call on another stream than the current one: memory
    that neither stream's work still uses."""
    a = Attention([40, 9], [1, 30], 4, 2, 64, 64, 16, 70)
    t = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
    free, table = ints([1, 2, 7]), ints([[3, -1, -1], [5, 6, -1]])
    cached, added = ints([15, 30]), ints([2, 2])
    stream = torch.cuda.Stream()
    on = stream.cuda_stream if raw else stream
    tables = [table.clone() for _ in range(9)]  # a call's, kept to the end
    each = iter(tables)

    def call():
        if operator == "attention":
            return pkg.shared_prefix_attention(a.q, a.kc, a.vc, *t, a.prefix,
                                               stream=on)
        return pkg.page_tables(cached, added, free, next(each), 16, 1000,
                               stream=on)[0]

    def work(big):
        for _ in range(10):
            big = big @ big * 1e-3

    torch.cuda.synchronize()
    want = call()
    torch.cuda.synchronize()
    want = want.clone()
    size = call().untyped_storage().nbytes()
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    # dropped before the call has run: not the next tensor's
    with torch.cuda.stream(stream):
        work(big)
    at = call().data_ptr()
    others = [torch.full((size,), 7, dtype=torch.uint8, device="cuda")
              for _ in range(3)]
    assert at not in [x.data_ptr() for x in others]
    torch.cuda.synchronize()
    assert all(bool((x == 7).all()) for x in others)
    # memory that the current stream's work still reads: not the call's
    del others
    last = torch.full((size,), 7, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    work(big)
    copy, at = last.clone(), last.data_ptr()
    del last
    got = call()
    assert got.data_ptr() != at
    torch.cuda.synchronize()
    assert bool((copy == 7).all()) and torch.equal(got, want)
    # the current stream's work with results that are dropped meanwhile
    got = call()
    torch.cuda.current_stream().wait_stream(stream)
    work(big)
    copy, at = got.clone(), got.data_ptr()
    del got
    with torch.cuda.stream(stream):
        others = [torch.full((size,), 7, dtype=torch.uint8, device="cuda")
                  for _ in range(3)]
    assert at not in [x.data_ptr() for x in others]
    torch.cuda.synchronize()
    assert torch.equal(copy, want)


def test_threads_on_one_stream(pkg, dev, monkeypatch):
    """Calls that two threads make on one stream take turns from the first of
    their launches to the last, on a buffer that no other operator has."""
    batches = [Attention([900, 40, 300 + s], [1, 2, 1], 8, 2, 64, 64, 16,
                         1500 + 900 * s, seed=s) for s in range(2)]
    want = [a.call(pkg).clone() for a in batches]
    x = torch.randn(64, 8192, device="cuda").half()
    w = torch.randn(8192, 256, device="cuda").half()
    product = pkg.matmul(x, w)
    torch.cuda.synchronize()
    real, inside, used, met = pkg.library(), [], [], []

    class Slow:
        """The library, with time for others before a call's launches."""

        def __getattr__(self, name):
            return getattr(real, name)

        def iree_mi355x_shared_prefix_attention_f16(self, args, ws, wsb, s):
            used.append((ws, wsb))
            inside.append(s)
            met.append(len(inside))
            time.sleep(0.01)
            st = real.iree_mi355x_shared_prefix_attention_f16(args, ws, wsb,
                                                              s)
            inside.pop()
            return st

    monkeypatch.setattr(pkg, "library", Slow)
    got, products, start = [[], []], [], threading.Barrier(3)

    def attend(t):
        start.wait()
        for _ in range(5):
            got[t].append(batches[t].call(pkg))

    def multiply():
        start.wait()
        for _ in range(50):
            products.append(pkg.matmul(x, w))

    threads = [threading.Thread(target=attend, args=(t,)) for t in range(2)]
    threads.append(threading.Thread(target=multiply))
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(used) == 10 and met == [1] * 10, met
    for g, o in zip(got, want):
        assert len(g) == 5 and all(torch.equal(x, o) for x in g)
    assert len(products) == 50
    assert all(torch.equal(p, product) for p in products)
    flat = [b for (_, _, layout), bufs in pkg._STREAM_WORKSPACES.items()
            if layout is None for b in bufs]
    for ws, wsb in used:
        assert all(ws + wsb <= b.data_ptr() or b.data_ptr() + b.numel() <= ws
                   for b in flat)


class Seen:
    """The library, which keeps the workspaces of attention calls."""

    def __init__(self, pkg):
        self.real, self.used = pkg.library(), []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def iree_mi355x_shared_prefix_attention_f16(self, args, ws, wsb, s):
        self.used.append((ws, wsb))
        return self.real.iree_mi355x_shared_prefix_attention_f16(args, ws,
                                                                 wsb, s)


def test_capture_on_another_stream(pkg, dev, monkeypatch):
    """A call on a stream forked from the capture, with other work captured
    beside it: what torch hands out then is not the call's workspace."""
    a = Attention([900, 40, 300], [1, 2, 1], 8, 2, 64, 64, 16, 1500)
    want = a.call(pkg).clone()
    t = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
    outs = [torch.empty_like(want) for _ in range(2)]
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    seen = Seen(pkg)
    monkeypatch.setattr(pkg, "library", lambda: seen)
    torch.cuda.synchronize()
    graph, beside = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        for o, stream in zip(outs, (side, side.cuda_stream)):
            pkg.shared_prefix_attention(a.q, a.kc, a.vc, *t, a.prefix, o,
                                        stream=stream)
            (ws, wsb) = seen.used[-1]
            for _ in range(3):
                x = torch.empty(wsb, dtype=torch.uint8, device="cuda")
                x.fill_(0x7f)
                beside.append(x)
        main.wait_stream(side)
    assert len(seen.used) == 2
    for ws, wsb in seen.used:
        assert ws and wsb and all(
            ws + wsb <= x.data_ptr() or x.data_ptr() + x.numel() <= ws
            for x in beside)
    for turn in range(4):
        for o in outs:
            o.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        eager = a.call(pkg)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs + [eager]), turn
        assert all(bool((x == 0x7f).all()) for x in beside)


def test_eager_call_beside_a_capture(pkg, dev, monkeypatch):
    """A call on a stream that is not captured while the current one is: the
    stream has no buffer yet and gets none, the call runs."""
    a = Attention([900, 40, 300], [1, 2, 1], 8, 2, 64, 64, 16, 1500)
    t = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
    o = torch.full((a.rows, 8, 64), 9.0, dtype=H, device="cuda")
    main, other = torch.cuda.Stream(), torch.cuda.Stream()
    monkeypatch.setattr(pkg, "_PAGED_WORKSPACES", {})
    monkeypatch.setattr(pkg, "_STREAM_WORKSPACES", {})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main,
                          capture_error_mode="thread_local"):
        x = torch.full((1000,), 3.0, device="cuda")
        pkg.shared_prefix_attention(a.q, a.kc, a.vc, *t, a.prefix, o,
                                    stream=other)
    torch.cuda.synchronize()
    a.check(o)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((x == 3).all())
    want = a.call(pkg)  # with a buffer: the same within the roundings
    a.check(want)


def hip(status):
    assert status == 0, status


@pytest.mark.parametrize("current", [False, True])
def test_capture_not_torch(pkg, dev, monkeypatch, current):
    """A stream captured through the HIP API, torch's current one or another:
    the call keeps no memory that torch gives to later tensors."""
    a = Attention([900, 40, 300], [1, 2, 1], 8, 2, 64, 64, 16, 1500)
    a.check(a.call(pkg))
    t = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
    o = torch.full((a.rows, 8, 64), 9.0, dtype=H, device="cuda")
    stream = torch.cuda.Stream()
    seen, lib = Seen(pkg), pkg.library()
    monkeypatch.setattr(pkg, "library", lambda: seen)
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    s = ctypes.c_void_p(stream.cuda_stream)
    held = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    with torch.cuda.stream(stream):  # memory of this stream to hand out
        mine = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    del held, mine
    torch.cuda.synchronize()
    hip(lib.hipStreamBeginCapture(s, 2))  # relaxed
    with torch.cuda.stream(stream if current else None):
        pkg.shared_prefix_attention(a.q, a.kc, a.vc, *t, a.prefix, o,
                                    stream=stream)
    hip(lib.hipStreamEndCapture(s, ctypes.byref(graph)))
    hip(lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0))
    assert seen.used == [(None, 0)]
    with torch.cuda.stream(stream):
        for turn in range(3):
            o.fill_(9.0)
            hip(lib.hipGraphLaunch(run, s))
            stream.synchronize()
            a.check(o)
    hip(lib.hipGraphExecDestroy(run))
    hip(lib.hipGraphDestroy(graph))


def test_captured_step(pkg, dev):
    """Tables, rows and attention of a step in one graph, whose replays read
    what its inputs hold then; eager steps between give the same."""
    page, pages, width, heads, hk, d = 16, 40, 80, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    start = ints([[0, 1] + [-1] * (width - 2), [2] + [-1] * (width - 1)])

    def state():
        return {"cached": ints([20, 9]), "added": ints([1, 3]),
                "free": ints(range(10, 20)), "table": start.clone(),
                "kc": torch.zeros(pages, hk, page, d, dtype=H, device="cuda"),
                "vc": torch.zeros(pages, hk, page, d, dtype=H, device="cuda"),
                "kv": torch.zeros(6, hk, d, dtype=H, device="cuda"),
                "q": torch.zeros(6, heads, d, dtype=H, device="cuda"),
                "o": torch.zeros(6, heads, d, dtype=H, device="cuda")}

    def step(t):
        starts, lengths, slots, needed = pkg.page_tables(
            t["cached"], t["added"], t["free"], t["table"], page, 6)
        pkg.append_kv(t["kv"], t["kv"], t["kc"], t["vc"], slots)
        pkg.shared_prefix_attention(
            t["q"], t["kc"], t["vc"], starts, lengths, t["table"],
            ints_none, 0, t["o"])
        return lengths, needed

    ints_none = torch.empty(0, dtype=I32, device="cuda")
    captured, eager = state(), state()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(state())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        lengths, needed = step(captured)
    for added in ([1, 3], [4, 0], [2, 4], [0, 0], [1, 1]):
        q, kv = (torch.randn(6, n, d, generator=g).half().cuda()
                 for n in (heads, hk))
        for t in (captured, eager):
            t["added"].copy_(ints(added))
            t["q"].copy_(q)
            t["kv"].copy_(kv)
        graph.replay()
        their_lengths, their_need = step(eager)
        torch.cuda.synchronize()
        for n in ("table", "kc", "vc", "o"):
            assert torch.equal(captured[n], eager[n]), n
        assert torch.equal(lengths, their_lengths)
        assert torch.equal(needed, their_need)
        used = int(needed)
        for t, n in ((captured, lengths), (eager, their_lengths)):
            t["cached"].copy_(n)
            t["free"].copy_(t["free"].roll(-used))


# Every head-dim bucket, narrow and wide tiles, rows joined by one group and
# by several (up to 8192 rows of all heads).
@pytest.mark.parametrize("added,heads,hk,d,dv", [
    ([1, 2, 1], 4, 2, 64, 64), ([1, 2, 40], 4, 2, 64, 64),
    ([1, 2, 40], 8, 2, 96, 96), ([300, 1, 20], 32, 4, 128, 128),
    ([1, 2, 40], 4, 2, 192, 128), ([1, 2, 1], 4, 2, 256, 256),
    ([300, 1, 20], 32, 4, 256, 256)])
@pytest.mark.parametrize("prefix", [0, 1500])
def test_attention_nan_parts(pkg, dev, added, heads, hk, d, dv, prefix):
    """A row whose scores are all NaN, in every part or in one kind's, is NaN
    where its tiles are split as well, and does nothing to other rows."""
    print(f"nan {added} {heads} {hk} {d} {prefix}", flush=True)
    a = Attention([1040, 9, 300], added, heads, hk, d, dv, 16, prefix, pad=1,
                  spare=columns(16))
    want = a.call(pkg).clone()
    assert bool(want.isfinite().all())
    q = a.q.clone()
    rows = sum(added)
    ill = torch.zeros(a.rows, heads, dtype=torch.bool, device="cuda")
    for row, head in ((0, 1), (added[0], heads - 1), (rows - 1, 0)):
        a.q[row, head] = NAN
        ill[row, head] = True
    o = a.call(pkg)
    assert bool(o[ill].isnan().all()) and torch.equal(o[~ill], want[~ill])
    # every key of the last KV head's prefix, or of request 0's own
    a.q = q
    group = heads // hk
    pages = a.prefix_pages if prefix else a.table[0][:up(a.lengths[0], 16)]
    a.kc[torch.tensor(pages, device="cuda"), hk - 1] = NAN
    ill[:] = False
    ill[:rows if prefix else added[0], heads - group:] = True
    o = a.call(pkg)
    assert bool(o[ill].isnan().all()) and torch.equal(o[~ill], want[~ill])


def abi(pkg, a, o):
    """The C-ABI's arguments of a call, and the tables to keep."""
    args = pkg.PagedAttentionArgs(
        q=a.q.data_ptr(), o=o.data_ptr(), rows=a.rows, heads=a.heads,
        batch=len(a.added), table_width=a.width, table_stride=a.width,
        prefix_length=a.prefix, scale=a.scale)
    keep = [ints(x) for x in (a.starts, a.lengths, a.table, a.prefix_pages)]
    for n, t in zip(("row_starts", "lengths", "block_table", "prefix_pages"),
                    keep):
        setattr(args, n, t.data_ptr())
    c = args.cache
    c.k, c.v = a.kc.data_ptr(), a.vc.data_ptr()
    c.pages, c.kv_heads, c.page_size, c.head_dim = a.kc.shape
    c.head_dim_v = a.dv
    c.k_strides[:], c.v_strides[:] = a.kc.stride()[:3], a.vc.stride()[:3]
    args.q_strides[:], args.o_strides[:] = a.q.stride()[:2], o.stride()[:2]
    return args, keep


# row starts (a pattern and how often), heads, kv heads, d, dv, prefix
STARTS = [([0, 1], 500, 16, 1, 64, 64, 32768),
          ([0, 4], 128, 32, 8, 64, 64, 32768),
          ([0, 4], 2048, 32, 8, 64, 64, 4096),
          ([0, 1], 500, 16, 1, 256, 256, 32768),
          ([0, 4], 128, 32, 8, 192, 128, 32768),
          ([0, 3, 1, 2, 0, 4], 300, 32, 8, 96, 96, 9000)]


@pytest.mark.parametrize("starts,times,heads,hk,d,dv,prefix", STARTS)
def test_attention_row_starts_guarded(pkg, dev, starts, times, heads, hk, d,
                                      dv, prefix):
    """Many requests whose starts do not ascend count the rows again and again:
    nothing outside o and the workspace is written, and the parts hold a batch
    of requests in order afterwards."""
    page, rows = 16, max(starts)
    a = Attention([5, 40, 9, 2], [rows, 0, 0, 0], heads, hk, d, dv, page, 64,
                  spare=3)
    a.prefix_pages = (a.prefix_pages * up(prefix, 64))[:up(prefix, page)]
    a.prefix = prefix
    in_order = a.starts, a.table, a.lengths, a.added
    batch = len(starts) * times
    a.starts = starts * times + [0]
    a.table = [a.table[0]] * batch
    a.lengths = [7] * batch
    a.added = [0] * batch
    out = torch.full((3 * rows, heads, dv), 9.0, dtype=H, device="cuda")
    o = out[rows:2 * rows]
    lib, s = pkg.library(), torch.cuda.current_stream().cuda_stream
    args, keep = abi(pkg, a, o)
    need = lib.iree_mi355x_shared_prefix_attention_workspace_bytes(
        ctypes.byref(args))
    head, guard = 256 << 10, 64 << 20
    assert need > head
    ws = torch.full((need + guard,), 0xA5, dtype=torch.uint8, device="cuda")
    print(f"starts {starts} x {times}, {heads} {hk} {d} {prefix}", flush=True)
    for size in (need, 0):
        assert lib.iree_mi355x_shared_prefix_attention_f16(
            ctypes.byref(args), ws.data_ptr() if size else None, size,
            s) == pkg.OK
        torch.cuda.synchronize()
        assert bool((ws[need:] == 0xA5).all()) and bool(
            (ws[:head] == 0xA5).all())
        assert bool((out[:rows] == 9).all()) and bool(
            (out[2 * rows:] == 9).all())
    a.starts, a.table, a.lengths, a.added = in_order
    args, keep = abi(pkg, a, o)
    assert lib.iree_mi355x_shared_prefix_attention_workspace_bytes(
        ctypes.byref(args)) <= need
    assert lib.iree_mi355x_shared_prefix_attention_f16(
        ctypes.byref(args), ws.data_ptr(), need, s) == pkg.OK
    a.check(o)


# ------------------------------------------------------------- all together --

def test_steps(pkg, dev):
    """A batch behind a prefix over several steps: tables, rows appended, and
    attention, against one contiguous cache for each request."""
    g = torch.Generator().manual_seed(5)
    heads, hk, d, page, prefix, batch = 6, 2, 64, 16, 37, 4
    pages, width = 60, 8
    kc, vc = (torch.full((pages, hk, page, d), NAN, dtype=H, device="cuda")
              for _ in range(2))
    free = torch.randperm(pages, generator=g).to(I32).cuda()
    table = torch.full((batch + 1, width), -1, dtype=I32, device="cuda")
    past = [[] for _ in range(batch + 1)]  # (k, v) rows, the prefix last
    cached = torch.zeros(batch + 1, dtype=I32, device="cuda")
    steps = [[0, 0, 0, 0, prefix], [20, 1, 0, 33, 0], [1, 1, 1, 1, 0],
             [1, 0, 5, 1, 0], [1, 1, 1, 17, 0], [1, 1, 1, 1, 0]]
    for added in steps:
        rows = sum(added) + 2
        k, v = (torch.randn(rows, hk, d, generator=g).half().cuda()
                for _ in range(2))
        q = torch.randn(rows, heads, d, generator=g).half().cuda()
        starts, lengths, slots, needed = pkg.page_tables(
            cached, ints(added), free, table, page, rows)
        pkg.append_kv(k, v, kc, vc, slots)
        at = 0
        for b, n in enumerate(added):
            past[b] += [(k[at + i], v[at + i]) for i in range(n)]
            at += n
        free, cached = free[int(needed):], lengths
        if added[batch]:
            continue
        o = pkg.shared_prefix_attention(
            q, kc, vc, starts[:batch + 1], lengths[:batch], table[:batch],
            table[batch], prefix)
        at = 0
        for b, n in enumerate(added[:batch]):
            if not n:
                continue
            seq = past[batch] + past[b]
            keys = torch.stack([x for x, _ in seq], 1)[None]
            vals = torch.stack([x for _, x in seq], 1)[None]
            hidden = torch.zeros(n, len(seq), dtype=H, device="cuda")
            for i in range(n):
                hidden[i, len(seq) - n + i + 1:] = -INF
            want = pkg.attention(
                q[at:at + n].transpose(0, 1)[None], keys, vals, causal=False,
                mask=hidden)[0].transpose(0, 1)
            got = o[at:at + n]
            # either is within 3 f16 roundings of values up to max |v| (see
            # Attention), an eighth of one more for the 32-bit sums
            assert (got.float() - want.float()).abs().max() \
                <= 6.25 * 2 ** -11 * vals.abs().max().float()
            at += n
