"""Packed rows on the GPU: rotary positions, the masks of drafted trees,
attention of trees over a paged cache, attention of whole sequences, and a
step of them in turn.

Whole numbers are compared for equality with a plain loop, the rest with the
definition in 64 bits, within bounds that count the kernels' roundings.
"""
import math

import pytest
import torch

from test_paged_gpu import Attention, ints, up

pytestmark = pytest.mark.gpu
H, F, D, I32 = torch.float16, torch.float32, torch.float64, torch.int32
NAN, INF = float("nan"), float("inf")


# ------------------------------------------------------------------- rotary --

def turned(x, positions, frequencies, sections, interleaved):
    """(y, bound). The kernel rounds y to f16 (2^-11 of it, or 2^-25 where it
    is subnormal). Its turn is a product of three 64-bit roundings and the
    reference's angle one of one: 2^-51 of the angle, at most; the part of a turn
    is rounded to 32 bits (pi 2^-25), the sine and cosine are off by two units of
    2^-24 and the three 32-bit operations by 2^-24 each: 2^-21 of |x1| + |x2|
    covers them."""
    x = x.double().cpu()
    positions = positions.reshape(-1, x.shape[0])
    y, bound = x.clone(), torch.zeros_like(x)
    half = frequencies.numel()
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(half):
        t = positions[axis[i]].double().cpu() * float(frequencies[i])
        c, s, t = t.cos()[:, None], t.sin()[:, None], t.abs()[:, None]
        at = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        x1, x2 = x[..., at[0]], x[..., at[1]]
        y[..., at[0]], y[..., at[1]] = x1 * c - x2 * s, x2 * c + x1 * s
        for a in at:
            bound[..., a] = (2 ** -11 * y[..., a].abs() + 2 ** -25 + (
                x1.abs() + x2.abs()) * (2 ** -21 + 2 ** -51 * t))
    return y, bound


def close(got, y, bound):
    off = (got.double().cpu() - y).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


ROTARY = [
    # rows, heads, kv heads, dim, sections
    (1, 1, 1, 2, (1,)), (3, 4, 0, 8, (4,)), (64, 32, 8, 128, (64,)),
    (37, 9, 3, 64, (8, 12, 12)), (5, 6, 2, 80, (10, 0, 30)),
    (130, 3, 1, 96, (8, 8, 4, 4)), (7, 5, 5, 256, (128,)),
    (33, 2, 2, 40, (3, 7)), (9, 3, 3, 33, (5, 6)), (17, 2, 1, 24, ()),
    (501, 1, 1, 16, (8,))]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary(pkg, dev, shape, interleaved):
    rows, h, hk, d, sections = shape
    print(f"rotary {shape} {interleaved}", flush=True)
    g = torch.Generator().manual_seed(rows + d)
    sections = sections or (0,)
    half = sum(sections)
    q = torch.randn(rows, h, d, generator=g).half().cuda()
    k = torch.randn(rows, hk, d, generator=g).half().cuda() if hk else None
    f = (10000.0 ** -(torch.arange(half) / max(half, 1))).float().cuda()
    top = 2 ** 31 - 1
    pos = torch.randint(-50, 100000, (len(sections), rows), generator=g)
    pos[0, 0], pos[-1, -1] = top, -top - 1
    pos = (pos[0] if len(sections) == 1 else pos).int().cuda()
    args = dict(sections=sections, interleaved=interleaved)
    qo, ko = pkg.rotary(q, k, pos, f, **args)
    want_q = turned(q, pos, f, sections, interleaved)
    close(qo, *want_q)
    assert qo.is_contiguous() and qo.dtype is H
    if hk:
        want_k = turned(k, pos, f, sections, interleaved)
        close(ko, *want_k)
    else:
        assert ko is None
    # views of one projection's rows, odd strides, in place
    for pad in (8, 3, 1):
        buf = torch.full((rows, (h + hk) * d + pad), 5.0, dtype=H,
                         device="cuda")
        qv = buf[:, :h * d].unflatten(1, (h, d))
        qv.copy_(q)
        kv = None
        if hk:
            kv = buf[:, h * d:(h + hk) * d].unflatten(1, (hk, d))
            kv.copy_(k)
        q2, k2 = pkg.rotary(qv, kv, pos, f, q_out=qv, k_out=kv, **args)
        assert q2 is qv and k2 is kv
        assert torch.equal(qv, qo) and (not hk or torch.equal(kv, ko))
        assert bool((buf[:, (h + hk) * d:] == 5).all())
    # heads first in memory, an output beside guards, positions apart
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.full((rows, h, d + 9), 5.0, dtype=H, device="cuda")
    far = torch.stack([pos, pos]) if pos.dim() == 1 else torch.cat(
        [pos, pos], 1)[:, :rows]
    q3, _ = pkg.rotary(qt, None, far[0] if pos.dim() == 1 else far, f,
                       q_out=out[..., 1:d + 1], **args)
    assert torch.equal(q3, qo)
    assert bool((out[..., 0] == 5).all() and (out[..., d + 1:] == 5).all())


def test_rotary_empty(pkg, dev):
    q = torch.zeros(0, 4, 16, dtype=H, device="cuda")
    f = torch.ones(8, device="cuda")
    qo, ko = pkg.rotary(q, q[:, :1], ints([]).reshape(0), f)
    assert qo.shape == (0, 4, 16) and ko.shape == (0, 1, 16)
    q = torch.zeros(3, 0, 16, dtype=H, device="cuda")
    assert pkg.rotary(q, None, ints([1, 2, 3]), f)[0].shape == (3, 0, 16)


def test_rotary_far_positions(pkg, dev):
    """Whole turns leave the values, half turns their negatives, however far."""
    q = torch.randn(4, 2, 16, device="cuda").half()
    f = torch.full((8,), math.pi, dtype=F, device="cuda")
    pos = ints([0, 2 ** 24 + 1, 10 ** 9, 2 ** 31 - 1])
    close(pkg.rotary(q, None, pos, f)[0], *turned(q, pos, f, (8,), False))


# -------------------------------------------------------------- tree masks --

def signed(word):
    word &= 0xffffffff
    return word - (1 << 32) if word >> 31 else word


def plain_masks(parents, starts, words, rows):
    masks, depths = [[0] * words for _ in range(rows)], [0] * rows
    for first, end in zip(starts, starts[1:]):
        bits = []
        for i in range(end - first):
            p = parents[first + i]
            p = p if 0 <= p < i else -1
            bits.append(1 << i | (bits[p] if p >= 0 else 0))
            depths[first + i] = depths[first + p] + 1 if p >= 0 else 0
            masks[first + i] = [signed(bits[i] >> 32 * w)
                                for w in range(words)]
    return masks, depths


@pytest.mark.parametrize("added", [
    [1], [0], [], [5, 0, 7], [64, 63, 65, 128, 129], [300, 1, 40],
    [3] * 200, [1000]])
@pytest.mark.parametrize("words", [1, 2, 9])
@pytest.mark.parametrize("kind", ["any", "chain", "near", "wrong"])
def test_tree_masks(pkg, dev, added, words, kind):
    print(f"masks {added[:5]} {words} {kind}", flush=True)
    g = torch.Generator().manual_seed(len(added) * 7 + words)
    pad = 5
    rows, parents = sum(added) + pad, []
    for n in added:
        for i in range(n):
            far = int(torch.randint(0, i + 1, (1,), generator=g))
            parents.append({"any": far - 1, "chain": i - 1,
                            "near": i - 1 - min(far, 3) if i else -1,
                            "wrong": far * 3 - 5}[kind])
    parents += [0] * pad
    starts = [sum(added[:b]) for b in range(len(added) + 1)]
    masks, depths = pkg.tree_masks(ints(parents), ints(starts), words)
    want = plain_masks(parents, starts, words, rows)
    assert masks.dtype is I32 and depths.dtype is I32
    assert masks.tolist() == want[0] and depths.tolist() == want[1]


def test_tree_masks_bounds(pkg, dev):
    """Parents at the type's ends; starts that do not ascend or lie outside
    the rows write nothing outside; no rows."""
    top = 2 ** 31 - 1
    masks, depths = pkg.tree_masks(ints([top, -top - 1, 1, 2, 0]),
                                   ints([0, 5]), 1)
    assert masks[:, 0].tolist() == [1, 2, 6, 14, 17]
    assert depths.tolist() == [0, 0, 1, 2, 1]
    buf = torch.zeros(300, dtype=I32, device="cuda")
    for starts in ([0, 200, 100, 300], [-5, 400], [top, -top - 1, 7],
                   [300, 0]):
        masks, _ = pkg.tree_masks(buf, ints(starts), 3)
        torch.cuda.synchronize()
    masks, depths = pkg.tree_masks(buf[:0], ints([0, 0]), 2)
    assert masks.shape == (0, 2) and depths.shape == (0,)


# ----------------------------------------------------------- tree attention --

class Tree(Attention):
    """Attention whose rows see only some of their request's new tokens."""

    def __init__(self, *args, words=1, seed=0, **kw):
        super().__init__(*args, seed=seed, **kw)
        g = torch.Generator().manual_seed(seed + 1)
        self.words = words
        self.parents = []
        for n in self.added:
            for i in range(n):
                back = int(torch.randint(0, min(i + 1, 5), (1,), generator=g))
                self.parents.append(i - 1 - back)
        self.parents += [0] * (self.rows - len(self.parents))
        self.masks = torch.tensor(
            plain_masks(self.parents, self.starts, words, self.rows)[0],
            dtype=I32).reshape(self.rows, words)

    def call(self, pkg, o=None, masks=None, **kw):
        if o is None:
            o = torch.full((self.rows, self.heads, self.dv), 9.0, dtype=H,
                           device="cuda")
        out = pkg.tree_attention(
            self.q, self.kc, self.vc, ints(self.starts), ints(self.lengths),
            ints(self.table).reshape(len(self.added), self.width),
            self.masks.cuda() if masks is None else masks,
            ints(self.prefix_pages), self.prefix, o, **kw)
        assert out is o
        return o

    def expected(self):
        kc, vc = self.kc.double().cpu(), self.vc.double().cpu()
        q = self.q.double().cpu()
        o = torch.full((self.rows, self.heads, self.dv), NAN, dtype=D)
        bound = o.clone()
        group, flat = self.heads // self.hk, {}
        self.kcpu, self.vcpu = kc, vc
        for b, a in enumerate(self.added):
            first, n = self.starts[b], self.lengths[b]
            for g in range(self.hk if a else 0):
                k, v, there = self.keys(b, g)
                node = torch.arange(len(k)) - self.prefix - (n - a)
                for i in range(a):
                    mask = self.masks[first + i].tolist()
                    bit = torch.tensor(
                        [j < 0 or j <= i and (
                            j >= 32 * self.words
                            or mask[j // 32] >> (j % 32) & 1 == 1)
                         for j in node.tolist()], dtype=torch.bool)
                    sees = there & (bit | (torch.arange(len(k))
                                           < self.prefix))
                    for h in range(g * group, (g + 1) * group):
                        o[first + i, h], bound[first + i, h] = attended(
                            q[first + i, h], k[sees], v[sees], self.scale)
        return o, bound


def attended(row, k, v, scale, out=2 ** -11):
    """One row's result and how far a kernel's may be off it, as Attention
    derives it; `out`: the result's rounding."""
    if not len(k):
        return 0.0, 0.0
    s = k @ row * scale
    p = torch.softmax(s, 0)
    r = p @ v
    big = (k.abs() @ row.abs()).max() * abs(scale)
    spread, n = p @ v.abs() + r.abs(), len(k)
    far = (out * r.abs() + 2 ** -11 * spread + 2 ** -25
           + n * 2 ** -25 * (v.abs().amax(0) + r.abs())
           + (n + (len(row) + 8) * big) * 2 ** -24 * spread)
    return r, 1.02 * far


TREES = [
    # cached, added, heads, kv heads, d, dv, page, prefix, words
    ([5], [1], 1, 1, 8, 8, 16, 0, 1),
    ([100], [8], 9, 3, 64, 64, 16, 0, 1),
    ([0], [7], 4, 1, 64, 64, 16, 0, 1),
    ([3, 0, 40, 31], [5, 1, 0, 9], 8, 2, 128, 128, 16, 64, 1),
    ([33, 31, 64, 7], [31, 32, 33, 64], 4, 2, 64, 64, 7, 0, 2),
    ([100, 257], [40, 70], 8, 2, 128, 128, 16, 0, 1),
    ([70, 3], [33, 16], 16, 2, 96, 96, 24, 130, 2),
    ([10, 0, 200], [2, 17, 40], 4, 1, 192, 128, 8, 100, 2),
    ([63, 64], [9, 20], 2, 2, 256, 256, 64, 31, 1),
    ([1000], [12], 8, 2, 64, 64, 16, 2000, 1),
    ([1500, 4], [70, 64], 4, 2, 128, 128, 64, 0, 3),
    ([20], [130], 2, 1, 40, 24, 5, 0, 2)]


@pytest.mark.parametrize("shape", TREES)
def test_tree_attention(pkg, dev, shape):
    cached, added, heads, hk, d, dv, page, prefix, words = shape
    print(f"tree {shape}", flush=True)
    for spare in (1, 90):  # a table that takes parts
        t = Tree(cached, added, heads, hk, d, dv, page, prefix, pad=3,
                 spare=spare, words=words, seed=len(cached) + d)
        t.check(t.call(pkg))


def test_tree_attention_of_chains(pkg, dev):
    """Masks of chains are what shared_prefix_attention computes, both within the
    definition's bounds (not the same bits: a block in which masks are looked at
    rounds s * scale before it subtracts the maximum, another block does both in
    one rounding); a mask's bits of later tokens are not looked at."""
    for added in ([3, 1, 5], [40, 70, 2], [100]):
        t = Tree([90, 700, 31][:len(added)], added, 8, 2, 64, 64, 16, 70)
        t.parents = [i - 1 for n in added for i in range(n)]
        t.words = up(max(added), 32)
        t.masks = torch.tensor(plain_masks(t.parents, t.starts, t.words,
                                           t.rows)[0], dtype=I32)
        t.check(Attention.call(t, pkg))
        got = t.call(pkg)
        t.check(got)
        ones = torch.full_like(t.masks, -1).cuda()
        assert torch.equal(t.call(pkg, masks=ones), got)


def test_tree_attention_masks_that_leave_nothing(pkg, dev):
    """A row whose mask is empty sees the cache alone, or nothing: 0."""
    for cached, prefix in ((0, 0), (50, 0), (0, 33)):
        for n in (4, 60):
            t = Tree([cached], [n], 4, 2, 64, 64, 16, prefix, words=2)
            t.masks[0] = 0
            t.masks[n - 1] = 0
            want = t.check(t.call(pkg))
            if not cached + prefix:
                assert bool((want[0] == 0).all())
    # fewer tokens than rows: the first nodes are not in the pages
    t = Tree([0], [40], 4, 2, 64, 64, 16, 20, words=2)
    t.lengths = [7]
    t.check(t.call(pkg))


def test_tree_attention_strided_masks(pkg, dev):
    t = Tree([90, 7], [33, 40], 8, 2, 128, 128, 16, 0, words=2)
    buf = torch.full((t.rows, 7), -1, dtype=I32, device="cuda")
    buf[:, 3:5] = t.masks.cuda()
    t.check(t.call(pkg, masks=buf[:, 3:5]))


# --------------------------------------------------------- packed attention --

class Packed:
    """Packed sequences of `added` queries and `keys` keys, their definition in
    64 bits and its bound."""

    def __init__(self, added, heads, hk, d, dv, keys=None, causal=True, pad=0,
                 fused=False, seed=0, heads_first=False):
        g = torch.Generator().manual_seed(seed)
        self.added, self.keys = added, keys or added
        self.causal, self.apart = causal, keys is not None
        self.heads, self.hk, self.d, self.dv = heads, hk, d, dv
        self.rows = sum(added) + pad
        n = sum(self.keys) + pad

        def rows_of(rows, h, dim):
            x = torch.randn(rows, h, dim, generator=g).half().cuda()
            if heads_first:
                return x.transpose(0, 1).contiguous().transpose(0, 1)
            return x

        if fused and not self.apart:
            x = rows_of(n, 1, heads * d + hk * (d + dv) + 8)[:, 0]
            q, k, v, _ = x.split([heads * d, hk * d, hk * dv, 8], 1)
            self.q, self.k, self.v = (
                q.unflatten(1, (heads, d)), k.unflatten(1, (hk, d)),
                v.unflatten(1, (hk, dv)))
        else:
            self.q = rows_of(self.rows, heads, d)
            self.k, self.v = rows_of(n, hk, d), rows_of(n, hk, dv)
        # rows of no sequence hold anything
        self.k[sum(self.keys):] = NAN
        self.v[sum(self.keys):] = NAN
        self.starts = [sum(added[:b]) for b in range(len(added) + 1)]
        self.key_starts = [sum(self.keys[:b]) for b in range(len(added) + 1)]

    def call(self, pkg, o=None, **kw):
        dtype = kw.pop("dtype", H)
        if o is None:
            o = torch.full((self.rows, self.heads, self.dv), 9.0, dtype=dtype,
                           device="cuda")
        out = pkg.packed_attention(
            self.q, self.k, self.v, ints(self.starts),
            ints(self.key_starts) if self.apart else None, o,
            causal=self.causal, **kw)
        assert out is o
        return o

    def check(self, got, scale=None):
        scale = self.d ** -0.5 if scale is None else scale
        out = torch.finfo(got.dtype).eps / 2
        group = self.heads // self.hk
        got = got.double()
        for b, (a, m) in enumerate(zip(self.added, self.keys)):
            r0, k0 = self.starts[b], self.key_starts[b]
            mine = got[r0:r0 + a]
            if not a:
                continue
            if not m:
                assert bool((mine == 0).all())
                continue
            sees = torch.ones(a, m, dtype=torch.bool, device="cuda")
            if self.causal:
                sees = sees.tril(m - a)
            for h in range(self.heads):
                q = self.q[r0:r0 + a, h].double()
                k = self.k[k0:k0 + m, h // group].double()
                v = self.v[k0:k0 + m, h // group].double()
                s = (q @ k.t() * scale).masked_fill(~sees, -INF)
                p = torch.softmax(s, 1).nan_to_num(0.0)  # rows that see none
                r, n = p @ v, sees.sum(1, keepdim=True)
                big = ((q.abs() @ k.abs().t()).masked_fill(~sees, 0.0)
                       .amax(1, keepdim=True) * abs(scale))
                spread = p @ v.abs() + r.abs()
                far = (out * r.abs() + 2 ** -11 * spread + 2 ** -25
                       + n * 2 ** -25 * (v.abs().amax(0) + r.abs())
                       + (n + (self.d + 8) * big) * 2 ** -24 * spread)
                off = (mine[:, h] - r).abs() - 1.02 * far
                assert bool((off <= 0).all()), (b, h, float(off.max()))
                none = n[:, 0] == 0
                assert bool((mine[none, h] == 0).all())
        assert bool((got[self.starts[-1]:] == 9).all()), "past the last"


PACKED = [
    # added, heads, kv heads, d, dv, keys
    ([1], 1, 1, 8, 8, None),
    ([37], 9, 3, 64, 64, None),
    ([5, 0, 1, 16, 17, 3], 4, 2, 64, 64, None),
    ([64, 128, 129, 63], 4, 4, 128, 128, None),
    ([300, 2, 77], 8, 2, 128, 128, None),
    ([70, 130, 200], 6, 1, 96, 96, None),
    ([100, 33], 3, 3, 80, 48, None),
    ([90, 200], 4, 1, 192, 128, None),
    ([1, 2, 3, 1], 4, 1, 192, 128, None),
    ([70, 9, 300], 2, 2, 256, 256, None),
    ([1, 1, 2], 2, 1, 256, 256, None),
    ([40, 150], 2, 1, 200, 232, None),
    ([200], 2, 2, 40, 24, None),
    # queries behind more keys, fewer keys than queries, none
    ([1, 1, 1], 8, 2, 128, 128, [900, 1, 65]),
    ([70, 3, 128], 4, 2, 64, 64, [1000, 700, 128]),
    ([100, 20, 7, 0], 4, 2, 64, 64, [30, 0, 3, 50]),
    ([20, 300], 2, 1, 256, 256, [400, 310])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", PACKED)
def test_packed(pkg, dev, shape, causal):
    added, heads, hk, d, dv, keys = shape
    print(f"packed {shape} {causal}", flush=True)
    p = Packed(added, heads, hk, d, dv, keys, causal, pad=3, seed=d)
    p.check(p.call(pkg))
    p.check(p.call(pkg, dtype=F))
    p = Packed(added, heads, hk, d, dv, keys, causal, pad=70, seed=d,
               fused=True, heads_first=keys is not None)
    p.check(p.call(pkg))


@pytest.mark.parametrize("added,heads,hk,d", [
    ([1500], 2, 2, 64),               # parts of many tiles
    ([1100], 8, 2, 128),
    ([2049], 16, 8, 128),             # whole tiles, heads on their XCDs
    ([700, 40, 1, 0, 900, 333], 24, 24, 64),   # and over all of them
    ([1, 2, 3, 4, 5, 6, 7] * 60, 6, 2, 96),
    ([16] * 130, 3, 3, 64), ([130] * 70, 2, 1, 128)])
def test_packed_many_tiles(pkg, dev, added, heads, hk, d):
    print(f"packed {added[:6]} {heads} {hk} {d}", flush=True)
    for causal in (True, False):
        p = Packed(added, heads, hk, d, d, causal=causal, pad=1, seed=d)
        p.check(p.call(pkg))


def test_packed_defaults(pkg, dev):
    p = Packed([70, 3], 4, 2, 64, 64)
    o = pkg.packed_attention(p.q, p.k, p.v, ints(p.starts))
    assert o.dtype is H and o.shape == (73, 4, 64) and o.is_contiguous()
    p.check(o)
    o = pkg.packed_attention(p.q, p.k, p.v, ints(p.starts), out_dtype=F,
                             scale=0.3)
    assert o.dtype is F
    p.check(o, scale=0.3)
    o = pkg.packed_attention(p.q, p.k, p.v, ints(p.starts), scale=-0.2)
    p.check(o, scale=-0.2)
    # no sequences, no rows
    o = torch.full((5, 4, 64), 9.0, dtype=H, device="cuda")
    pkg.packed_attention(p.q[:5], p.k[:5], p.v[:5], ints([0]), o=o)
    assert bool((o == 9).all())
    assert pkg.packed_attention(p.q[:0], p.k[:0], p.v[:0],
                                ints([0, 0])).shape == (0, 4, 64)
    # no keys at all
    o = pkg.packed_attention(p.q, p.k[:0], p.v[:0], ints(p.starts),
                             ints([0, 0, 0]))
    assert bool((o == 0).all())


def test_packed_output_views(pkg, dev):
    """Outputs in the columns of a wider buffer, at 16 and at 8 bytes, whole
    tiles and parts of f16 and f32: what lies beside them stays."""
    for added, heads, hk, d in (([70, 3], 4, 2, 64), ([1500], 2, 2, 64),
                                ([900], 2, 1, 128), ([9, 5], 2, 1, 40)):
        p = Packed(added, heads, hk, d, d)
        for dtype in (H, F):
            for pad, at in ((8, 0), (8, 8), (4, 4), (12, 4)):
                print(f"views {added} {dtype} {pad} {at}", flush=True)
                buf = torch.full((p.rows, heads, d + pad), 9.0, dtype=dtype,
                                 device="cuda")
                view = buf[..., at:at + d]
                p.check(p.call(pkg, view))
                assert bool((buf[..., :at] == 9).all()
                            and (buf[..., at + d:] == 9).all())
        with pytest.raises(pkg.MI355XError, match="aligned|multiples"):
            p.call(pkg, torch.zeros(p.rows, heads, d + 2, dtype=H,
                                    device="cuda")[..., 2:])


def test_packed_far_rows(pkg, dev):
    """Keys whose bytes pass 32 bits, in narrow and wide tiles and in parts."""
    stride, d, n = 1 << 24, 64, 140
    buf = torch.empty(stride * (n - 1) + 2 * d, dtype=H, device="cuda")
    k = buf.as_strided((n, 1, d), (stride, d, 1))
    v = buf[d:].as_strided((n, 1, d), (stride, d, 1))
    g = torch.Generator().manual_seed(3)
    for x in (k, v):
        x.copy_(torch.randn(n, 1, d, generator=g).half().cuda())
    for added, keys in (([140], None), ([2, 1], [5, 135]), ([60, 3], [7, 133])):
        print(f"far {added} {keys}", flush=True)
        p = Packed(added, 1, 1, d, d, keys)
        p.k, p.v = k, v
        p.check(p.call(pkg))
    # as the last of 6000 rows, in parts
    k, v = (torch.randn(6000, 1, d, generator=g).half().cuda()
            for _ in range(2))
    p = Packed([1, 40], 1, 1, d, d, [100, 5900])
    p.k, p.v = k, v
    p.check(p.call(pkg))


def test_packed_threads(pkg, dev):
    """Calls of several threads on one stream, each of two launches, keep
    their parts."""
    import threading
    calls = [Packed([1500 + 100 * i], 2, 2, 64, 64, seed=i) for i in range(4)]
    want = [p.call(pkg) for p in calls]
    got = [[] for _ in calls]

    def run(i):
        for _ in range(20):
            got[i].append(calls[i].call(pkg))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, p in enumerate(calls):
        p.check(want[i])
        assert len(got[i]) == 20
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_packed_ordered_tiles(pkg, dev):
    """More tiles than run at once, of requests of many lengths: ordered by
    their keys, each found once; and of more requests than lanes."""
    g = torch.Generator().manual_seed(11)
    for batch, lo, hi, heads, hk, causal in (
            (17, 200, 900, 24, 8, True), (64, 0, 700, 6, 6, True),
            (30, 1, 1000, 9, 3, False), (65, 100, 500, 8, 8, True),
            (2, 2000, 2600, 8, 8, True)):
        added = torch.randint(lo, hi, (batch,), generator=g).tolist()
        keys = [n + int(torch.randint(0, 300, (1,), generator=g))
                for n in added]
        keys[0] = 0
        print(f"ordered {batch} {heads} {hk}", flush=True)
        p = Packed(added, heads, hk, 64, 64, keys, causal, pad=2, seed=batch)
        p.check(p.call(pkg))


@pytest.mark.parametrize("batch,lo,hi,heads,hk,d,more", [
    (257, 0, 140, 2, 1, 64, None),    # one more than are counted
    (300, 0, 9, 2, 1, 256, 70),       # narrow tiles alone
    (320, 10, 60, 1, 1, 256, None),
    (700, 0, 40, 3, 1, 96, 90), (400, 1, 1, 8, 1, 128, 300),
    (4200, 0, 12, 1, 1, 64, None)])   # three rounds of 64
def test_packed_many_sequences(pkg, dev, batch, lo, hi, heads, hk, d, more):
    """More sequences than a workgroup counts, empty ones among them."""
    print(f"many {batch} {lo} {hi} {heads} {hk} {d} {more}", flush=True)
    g = torch.Generator().manual_seed(batch)

    def lengths(lo, hi):
        n = torch.randint(lo, hi + 1, (batch,), generator=g)
        # runs of sequences without rows, the first and the last among them
        n[:3], n[70:90], n[-2:] = lo, lo, lo
        return n.tolist()

    added = lengths(lo, hi)
    keys = lengths(0, more) if more else None
    p = Packed(added, heads, hk, d, d, keys, causal=batch % 200 != 0, pad=5,
               seed=d)
    p.check(p.call(pkg))


def test_packed_many_bad_starts(pkg, dev):
    """Starts of many sequences that do not ascend: nothing outside is
    written."""
    p = Packed([200, 100], 4, 2, 64, 64)
    top = 2 ** 31 - 1
    for rows in ([0, 300] * 200, [300, 0] * 200, [-5, top] * 150,
                 [300] * 301, [top] * 301, [0] * 301,
                 list(range(300, -1, -1))):
        print(f"starts {rows[:3]} {len(rows)}", flush=True)
        buf = torch.full((302, 4, 64), 9.0, dtype=H, device="cuda")
        pkg.packed_attention(p.q, p.k, p.v, ints(rows), None, buf[1:301])
        torch.cuda.synchronize()
        assert bool((buf[0] == 9).all() and (buf[301] == 9).all())


def test_packed_infinities(pkg, dev):
    """A NaN in a sequence's query or key stays in its rows; infinite scores of
    either sign are the formula's; other sequences' rows are not read."""
    p = Packed([100, 50, 140], 4, 2, 64, 64)
    clean = p.call(pkg)
    p.q[110, 1] = NAN
    p.k[160, 0] = NAN
    got = p.call(pkg)
    bad = got.isnan().all(2)
    want = torch.zeros_like(bad)
    want[110, 1] = True
    want[160:, :2] = True
    assert torch.equal(bad, want)
    assert torch.equal(got[~want], clean[~want])
    p = Packed([80], 2, 2, 64, 64)
    p.k[:, 0] = p.k[:, 0].abs()
    p.q[:, 0] = p.q[:, 0].abs()
    p.k[3, 0] = -INF  # scores of -inf: weight 0
    got = p.call(pkg)
    k = p.k.double().clone()
    s = (p.q[:, 0].double() @ k[:, 0].t() * 64 ** -0.5)
    s = s.masked_fill(~torch.ones(80, 80, device="cuda").bool().tril(), -INF)
    want = torch.softmax(s, 1) @ p.v[:, 0].double()
    assert (got[:, 0].double() - want).abs().max() < 0.01


def test_packed_bad_starts(pkg, dev):
    """Starts that do not ascend or lie outside the rows: rows hold anything,
    nothing outside the tensors is written."""
    p = Packed([200, 100], 4, 2, 64, 64)
    top = 2 ** 31 - 1
    for rows, keys in (([0, 300, 100, 300], [0, 200, 100, 300]),
                       ([-7, 150, top], [-top - 1, 100, top]),
                       ([300, 0, 300], [300, 0, 200]),
                       ([0, 300, 0, 300, 0, 300], [0, 300, 0, 300, 0, 300])):
        print(f"starts {rows} {keys}", flush=True)
        buf = torch.full((302, 4, 64), 9.0, dtype=H, device="cuda")
        pkg.packed_attention(p.q, p.k, p.v, ints(rows), ints(keys),
                             buf[1:301])
        torch.cuda.synchronize()
        assert bool((buf[0] == 9).all() and (buf[301] == 9).all())


# ---------------------------------------------------------------- the layer --

def test_a_step_of_trees(pkg, dev):
    """Drafted trees over a cache that a prompt has filled: masks, positions,
    rotation, rows appended, attention; against the same in 64 bits."""
    torch.manual_seed(5)
    h, hk, d, page = 8, 2, 64, 16
    prompts, added = [70, 33], [9, 20]
    f = (10000.0 ** -(torch.arange(32) / 32.0)).float().cuda()
    pages = sum(up(a + n, page) for a, n in zip(prompts, added))
    kc = torch.zeros(pages, hk, page, d, dtype=H, device="cuda")
    vc = torch.zeros_like(kc)
    free, table = ints(list(range(pages))), torch.full(
        (2, 6), -1, dtype=I32, device="cuda")

    def rows(n):
        return (torch.randn(n, h, d).half().cuda(),
                torch.randn(n, hk, d).half().cuda(),
                torch.randn(n, hk, d).half().cuda())

    # the prompts
    q, k, v = rows(sum(prompts))
    starts, lengths, slots, taken = pkg.page_tables(
        ints([0, 0]), ints(prompts), free, table, page, sum(prompts))
    pos = torch.cat([torch.arange(n) for n in prompts]).int().cuda()
    q1, k1 = pkg.rotary(q, k, pos, f)
    pkg.append_kv(k1, v, kc, vc, slots)
    o1 = pkg.packed_attention(q1, k1, v, starts)
    same = pkg.shared_prefix_attention(q1, kc, vc, starts, lengths, table)
    # the trees
    parents = [i - 1 - int(torch.randint(0, min(i + 1, 3), (1,)))
               for n in added for i in range(n)]
    tq, tk, tv = rows(sum(added))
    starts2, lengths2, slots2, _ = pkg.page_tables(
        ints(prompts), ints(added), free[int(taken):], table, page,
        sum(added))
    masks, depths = pkg.tree_masks(ints(parents), starts2)
    pos2 = depths + torch.repeat_interleave(ints(prompts), ints(added))
    q2, k2 = pkg.rotary(tq, tk, pos2.int(), f)
    pkg.append_kv(k2, tv, kc, vc, slots2)
    o2 = pkg.tree_attention(q2, kc, vc, starts2, lengths2, table, masks)
    # every node against its own path, as a sequence of its own
    row = 0
    for b, n in enumerate(prompts):
        at = sum(prompts[:b])
        for i in range(added[b]):
            path, j = [], i
            while j >= 0:
                path.insert(0, j)
                j = parents[row + j]
            idx = torch.tensor([row + j for j in path], device="cuda")
            xk = torch.cat([k1[at:at + n], k2[idx]])
            xv = torch.cat([v[at:at + n], tv[idx]])
            assert int(depths[row + i]) == len(path) - 1
            for hh in range(h):
                g = hh // (h // hk)
                want, far = attended(q2[row + i, hh].double(),
                                     xk[:, g].double(), xv[:, g].double(),
                                     d ** -0.5)
                assert bool(((o2[row + i, hh].double() - want).abs()
                             <= far).all())
        row += added[b]
    # the prompts' two forms: the same definition, either way within bounds
    for b, n in enumerate(prompts):
        at = sum(prompts[:b])
        for i in (0, 1, n - 1):
            for hh in range(h):
                g = hh // (h // hk)
                want, far = attended(q1[at + i, hh].double(),
                                     k1[at:at + i + 1, g].double(),
                                     v[at:at + i + 1, g].double(), d ** -0.5)
                for o in (o1, same):
                    assert bool(((o[at + i, hh].double() - want).abs()
                                 <= far).all())


def test_a_captured_step(pkg, dev):
    """Operators captured once and replayed with other lengths, parents and
    positions, eager work between the replays."""
    t = Tree([90, 40, 10], [20, 5, 33], 8, 2, 64, 64, 16, 0, pad=70, words=2,
             spare=4)
    p = Packed([60, 200, 9], 8, 2, 64, 64, pad=0)
    starts, lengths = ints(t.starts), ints(t.lengths)
    parents, table = ints(t.parents), ints(t.table)
    pstarts, pos = ints(p.starts), ints(list(range(p.rows)))
    f = torch.linspace(1, 0.1, 32, device="cuda")
    o = torch.zeros(t.rows, 8, 64, dtype=H, device="cuda")

    def step():
        masks, depths = pkg.tree_masks(parents, starts, 2)
        pkg.tree_attention(t.q, t.kc, t.vc, starts, lengths, table, masks,
                           o=o)
        q, k = pkg.rotary(p.q, p.k, pos, f)
        return masks, depths, pkg.packed_attention(q, k, p.v, pstarts), q

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for added, cut in (([20, 5, 33], [60, 200, 9]), ([1, 0, 40], [0, 269, 0]),
                       ([50, 17, 2], [100, 100, 69])):
        s = [0]
        for a in added:
            s.append(s[-1] + a)
        starts.copy_(ints(s))
        lengths.copy_(ints([c + a for c, a in zip([40, 41, 10], added)]))
        pstarts.copy_(ints([0, cut[0], cut[0] + cut[1], sum(cut)]))
        pos.add_(7)
        o.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        held = [x.clone() for x in out] + [o.clone()]
        o.fill_(9.0)
        fresh = step()
        for a, b in zip(held, list(fresh) + [o]):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_captured_parts(pkg, dev):
    """Calls of two launches in graphs of one stream, replayed beside eager calls
    with the stream's own buffer."""
    p = Packed([1500], 2, 2, 64, 64)
    t = Tree([1500, 40], [60, 9], 8, 2, 64, 64, 16, 0, words=2, spare=90)
    ps, ts = ints(p.starts), [ints(x) for x in (t.starts, t.lengths, t.table)]
    masks = t.masks.cuda()
    want_p, want_t = p.call(pkg), t.call(pkg)
    p.check(want_p)
    t.check(want_t)
    outs = []
    for _ in range(2):
        po = torch.zeros_like(want_p)
        to = torch.zeros_like(want_t)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pkg.packed_attention(p.q, p.k, p.v, ps, o=po)
            pkg.tree_attention(t.q, t.kc, t.vc, *ts, masks, o=to)
        outs.append((graph, po, to))
    for _ in range(3):
        for graph, po, to in outs:
            po.zero_()
            to.zero_()
            graph.replay()
            p.call(pkg)
            t.call(pkg)
        torch.cuda.synchronize()
        for _, po, to in outs:
            assert torch.equal(po, want_p) and torch.equal(to, want_t)


def test_another_stream(pkg, dev):
    """Calls that name another stream run in its order."""
    p = Packed([300, 41], 8, 2, 64, 64, pad=2)
    t = Tree([30, 90], [20, 9], 8, 2, 64, 64, 16, words=1)
    other = torch.cuda.Stream()
    want = p.call(pkg)
    f = torch.linspace(1, 0.1, 32, device="cuda")
    pos = ints(list(range(p.rows)))
    turned_q, _ = pkg.rotary(p.q, p.k, pos, f)
    masks, depths = pkg.tree_masks(ints(t.parents), ints(t.starts))
    starts, parents, tstarts = ints(p.starts), ints(t.parents), ints(t.starts)
    torch.cuda.synchronize()
    late = torch.zeros_like(p.q)
    with torch.cuda.stream(other):
        torch.cuda._sleep(20_000_000)
        late.copy_(p.q)
    got = pkg.packed_attention(late, p.k, p.v, starts, stream=other)
    q2, _ = pkg.rotary(late, p.k, pos, f, stream=other.cuda_stream)
    m2, d2 = pkg.tree_masks(parents, tstarts, stream=other)
    other.synchronize()
    n = p.starts[-1]
    assert torch.equal(got[:n], want[:n]) and torch.equal(q2, turned_q)
    assert torch.equal(m2, masks) and torch.equal(d2, depths)
