"""Tree attention of many requests behind a shared prefix: rows that share its
tiles and rows that do not, more requests than a wavefront has lanes, and lengths,
starts and tables that hold anything.

The definition in 64 bits and its bound are `Tree`'s.
"""
import ctypes

import pytest
import torch

from test_packed_gpu import Tree
from test_paged_gpu import ints

pytestmark = pytest.mark.gpu
H, I32 = torch.float16, torch.int32
TOP = 2 ** 31 - 1


def need(pkg, t):
    return pkg._paged_workspace_need(
        t.rows, len(t.added), t.heads, t.hk, t.d, t.dv, t.page, t.width,
        t.prefix)


MANY = [
    # requests, new tokens (cycled), heads, kv heads, d, dv, prefix, words
    # rows a KV head: 0, to 16 (narrow tiles), to 96 (the prefix's shared
    # tiles), above (tiles of their own)
    (65, (1, 4, 0, 5, 24, 25, 3), 4, 1, 64, 64, 300, 1),
    (130, (0, 1, 2, 24, 1, 30, 4, 12), 4, 1, 64, 64, 129, 1),
    (200, (1, 3, 0, 16, 2, 33), 3, 1, 96, 96, 200, 2),
    (100, (2, 9, 12, 0, 13, 1), 8, 1, 128, 128, 130, 1),
    # narrow tiles alone
    (70, (1, 5, 0, 17, 96, 2, 97), 1, 1, 256, 256, 140, 4),
    (129, (0, 16, 17, 1, 3), 1, 1, 192, 128, 65, 1),
    # wide tiles of longer keys
    (66, (20, 60, 0, 97, 1), 1, 1, 192, 128, 500, 4)]


@pytest.mark.parametrize("shape", MANY)
def test_trees_of_many_requests(pkg, dev, shape):
    batch, new, heads, hk, d, dv, prefix, words = shape
    print(f"trees {shape}", flush=True)
    added = [new[b % len(new)] for b in range(batch)]
    cached = [(7 * b) % 40 if b % 5 else 0 for b in range(batch)]
    t = Tree(cached, added, heads, hk, d, dv, 16, prefix, pad=2, spare=90,
             words=words, seed=batch)
    assert need(pkg, t) > 0
    got = t.call(pkg)
    t.check(got)
    # without a workspace: every request walks the prefix itself
    whole = torch.full_like(got, 9.0)
    assert raw(pkg, t, whole, None, 0) == pkg.OK
    t.check(whole)


def raw(pkg, t, o, workspace, bytes_, starts=None, lengths=None, table=None):
    """The C entry on a workspace of the caller's."""
    starts = ints(t.starts) if starts is None else starts
    lengths = ints(t.lengths) if lengths is None else lengths
    if table is None:
        table = ints(t.table).reshape(len(t.added), t.width)
    prefix, masks = ints(t.prefix_pages), t.masks.cuda()
    a = pkg.PagedAttentionArgs(
        q=t.q.data_ptr(), o=o.data_ptr(), row_starts=starts.data_ptr(),
        lengths=lengths.data_ptr(), block_table=table.data_ptr(),
        prefix_pages=prefix.data_ptr() if t.prefix else None, rows=t.rows,
        heads=t.heads, batch=lengths.numel(), table_width=table.shape[1],
        table_stride=table.stride(0), prefix_length=t.prefix,
        scale=t.d ** -0.5)
    c = a.cache
    c.k, c.v = t.kc.data_ptr(), t.vc.data_ptr()
    c.pages, c.kv_heads, c.page_size, c.head_dim = t.kc.shape
    c.head_dim_v = t.dv
    c.k_strides[:], c.v_strides[:] = t.kc.stride()[:3], t.vc.stride()[:3]
    a.q_strides[:], a.o_strides[:] = t.q.stride()[:2], o.stride()[:2]
    status = pkg.library().iree_mi355x_tree_attention_f16(
        ctypes.byref(a), masks.data_ptr(), t.words, masks.stride(0),
        workspace, bytes_, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()  # before its tables go
    return status


@pytest.mark.parametrize("batch,heads,hk,d,dv", [
    (6, 4, 1, 64, 64), (70, 4, 1, 64, 64), (6, 2, 1, 256, 256),
    (70, 6, 2, 128, 128), (70, 1, 1, 192, 128)])
def test_trees_of_bad_tables(pkg, dev, batch, heads, hk, d, dv):
    """Starts that do not ascend, lengths and pages of any value, behind a prefix
    that requests share: rows hold anything, but nothing beside the output or the
    workspace is written, whatever the workspace held, and the next call is
    right."""
    print(f"bad tables {batch} {heads} {d}", flush=True)
    added = [(1, 4, 20, 0, 30, 9)[b % 6] for b in range(batch)]
    t = Tree([17] * batch, added, heads, hk, d, dv, 16, 150, spare=90,
             words=1, seed=d)
    size, guard = need(pkg, t), 4096
    assert size > 0
    g = torch.Generator().manual_seed(batch)
    n = t.rows

    def some(lo, hi, count):
        return torch.randint(lo, hi, (count,), generator=g).tolist()

    right = t.table
    wild = [[x if x >= 0 else v for x, v in zip(row, some(-TOP, TOP, t.width))]
            for row in right]
    for starts, lengths, table in (
            ([0, n] * batch, t.lengths, right),
            ([n, 0] * batch, [TOP] * batch, right),
            ([-5, TOP] * batch, [-TOP - 1, TOP] * batch, wild),
            (some(0, n + 1, batch + 1), some(0, 2000, batch), wild),
            (sorted(some(0, n + 1, batch + 1)), some(-9, 90, batch), right),
            (some(-TOP, TOP, batch + 1), some(-TOP, TOP, batch), wild),
            (t.starts, [TOP] * batch, wild), (t.starts, [0] * batch, right),
            ([n] * (batch + 1), t.lengths, right),
            (list(range(batch + 1))[::-1], t.lengths, right)):
        for fill in (0, -1, 0x7f):
            buf = torch.full((n + 2, heads, dv), 9.0, dtype=H, device="cuda")
            ws = torch.full((size + 2 * guard,), fill, dtype=torch.int8,
                            device="cuda")
            ws[:guard] = ws[guard + size:] = 0x5a
            assert raw(pkg, t, buf[1:-1], ws.data_ptr() + guard, size,
                       ints(starts[:batch + 1]), ints(lengths[:batch]),
                       ints(table)) == pkg.OK
            assert bool((buf[0] == 9).all() and (buf[-1] == 9).all())
            assert bool((ws[:guard] == 0x5a).all()
                        and (ws[guard + size:] == 0x5a).all())
    buf = torch.full((n, heads, dv), 9.0, dtype=H, device="cuda")
    ws = torch.full((size,), 0x7f, dtype=torch.int8, device="cuda")
    assert raw(pkg, t, buf, ws.data_ptr(), size) == pkg.OK
    t.check(buf)
