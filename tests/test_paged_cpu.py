"""The paged KV cache without a GPU: what the Python operators and the C-ABI
refuse before anything is launched, and the workspace that attention asks
for."""
import ctypes

import pytest
import torch

H, I32 = torch.float16, torch.int32
FAKE = 1 << 20


def z(*shape, dtype=H):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape):
    return torch.zeros(*shape, dtype=I32)


# ---------------------------------------------------------------- operators --

def test_page_tables_checks(pkg):
    good = dict(cached=i(3), added=i(3), free_pages=i(5),
                block_table=i(3, 4), page_size=16, rows=7)

    def bad(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            pkg.page_tables(**{**good, **kw})

    bad("added", added=i(2))
    bad("int32", TypeError, added=torch.zeros(3, dtype=torch.int64))
    bad("int32", TypeError, free_pages=None)
    bad("block_table must be", block_table=i(2, 4))
    bad("2-D", block_table=i(12))
    bad("unit column", block_table=i(4, 3).t())
    bad("unit column", cached=i(6)[::2])
    bad("page_size", page_size=0)
    bad("rows", rows=-1)
    bad("device", TypeError)


def test_append_checks(pkg):
    good = dict(k=z(5, 2, 16), v=z(5, 2, 24), k_cache=z(3, 2, 8, 16),
                v_cache=z(3, 2, 8, 24), slots=i(5))

    def bad(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            pkg.append_kv(**{**good, **kw})

    bad("k must be", k=z(5, 2, 24))
    bad("v must be", v=z(4, 2, 24))
    bad("k must be a 3-D", TypeError, k=z(5, 32))
    bad("v_cache must be", v_cache=z(3, 2, 9, 24))
    bad("4-D f16", TypeError, k_cache=z(3, 2, 8, 16, dtype=torch.float32))
    bad("4-D f16", TypeError, k_cache=z(3, 2, 16, 8).transpose(2, 3))
    bad("slots", slots=i(6))
    bad("int32", TypeError, slots=torch.zeros(5, dtype=torch.int64))
    bad("device", TypeError)


def test_attention_checks(pkg):
    good = dict(q=z(5, 6, 16), k_cache=z(4, 2, 8, 16), v_cache=z(4, 2, 8, 24),
                row_starts=i(4), lengths=i(3), block_table=i(3, 2),
                prefix_pages=i(2), prefix_length=16)

    def bad(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            pkg.shared_prefix_attention(**{**good, **kw})

    bad("q must be", q=z(5, 6, 24))
    bad("multiple of 2 KV", q=z(5, 5, 16))
    bad("v_cache must be", v_cache=z(4, 3, 8, 24))
    bad("row_starts", row_starts=i(3))
    bad("block_table must be", block_table=i(4, 2))
    bad("int32", TypeError, lengths=torch.zeros(3))
    bad("prefix_pages hold", prefix_length=17)
    bad("needs prefix_pages", prefix_pages=None)
    bad("negative", prefix_length=-1)
    bad("o must be", o=z(5, 6, 16))
    bad("3-D f16", TypeError, o=z(5, 6, 24, dtype=torch.float32))
    bad("device", TypeError)
    bad("device", TypeError, prefix_pages=None, prefix_length=0)


# -------------------------------------------------------------------- C-ABI --

def tables(pkg, **kw):
    a = pkg.PageTablesArgs(
        cached=FAKE, added=FAKE, free_pages=FAKE, block_table=FAKE,
        row_starts=FAKE, lengths=FAKE, slots=FAKE, needed=FAKE, batch=3,
        free_count=5, page_size=16, table_width=4, table_stride=4, rows=7)
    for k, v in kw.items():
        setattr(a, k, v)
    return pkg.library().iree_mi355x_page_tables(ctypes.byref(a), None)


def test_page_tables_argument_errors(pkg):
    lib = pkg.library()
    assert lib.iree_mi355x_page_tables(None, None) == pkg.INVALID_ARGUMENT
    for kw in (dict(batch=-1), dict(rows=-1), dict(free_count=-1),
               dict(table_width=-1), dict(table_stride=-1),
               dict(page_size=0), dict(table_stride=3), dict(cached=None),
               dict(added=None), dict(free_pages=None),
               dict(block_table=None), dict(row_starts=None),
               dict(lengths=None), dict(slots=None), dict(needed=None)):
        assert tables(pkg, **kw) == pkg.INVALID_ARGUMENT, kw
        assert "page_tables" in pkg.last_error()
    for kw in (dict(batch=1 << 31), dict(rows=1 << 31),
               dict(page_size=1 << 31), dict(table_width=1 << 31),
               dict(table_stride=1 << 60)):
        assert tables(pkg, **kw) == pkg.UNSUPPORTED, kw
    assert tables(pkg, slots=FAKE + 2) == pkg.MISALIGNED


def cache(pkg, **kw):
    c = pkg.KvCache(k=FAKE, v=FAKE, pages=4, page_size=16, kv_heads=2,
                    head_dim=64, head_dim_v=64)
    c.k_strides[:] = c.v_strides[:] = [2 * 16 * 64, 16 * 64, 64]
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


CACHE_ERRORS = [
    (dict(pages=-1), "INVALID_ARGUMENT"), (dict(k=None), "INVALID_ARGUMENT"),
    (dict(page_size=0), "INVALID_ARGUMENT"),
    (dict(kv_heads=-1), "INVALID_ARGUMENT"),
    (dict(head_dim=60), "UNSUPPORTED"), (dict(head_dim_v=264), "UNSUPPORTED"),
    (dict(head_dim=0), "UNSUPPORTED"),
    (dict(pages=1 << 28), "UNSUPPORTED"), (dict(k=FAKE + 8), "MISALIGNED"),
    (dict(k_strides=[2048, 1024, 60]), "MISALIGNED"),
    (dict(v_strides=[2048, 1024, 56]), "INVALID_ARGUMENT"),
    (dict(v_strides=[-8, 1024, 64]), "INVALID_ARGUMENT"),
    # a head's rows over 64 GiB: 3 pages of 16 GiB reach 48, of 24 GiB 72
    (dict(k_strides=[3 << 32, 1024, 64]), "UNSUPPORTED"),
    (dict(k_strides=[1 << 62, 1024, 64]), "UNSUPPORTED"),
]


@pytest.mark.parametrize("kw,status", CACHE_ERRORS)
def test_cache_argument_errors(pkg, kw, status):
    c, want = cache(pkg, **kw), getattr(pkg, status)
    st = (ctypes.c_int64 * 2)(128, 64)
    assert pkg.library().iree_mi355x_append_kv_f16(
        ctypes.byref(c), FAKE, FAKE, 3, st, st, FAKE, None) == want
    assert "append_kv" in pkg.last_error()
    assert attend(pkg, c) == want
    assert "shared_prefix_attention" in pkg.last_error()


def test_append_argument_errors(pkg):
    lib, c = pkg.library(), cache(pkg)

    def call(c=c, k=FAKE, v=FAKE, rows=3, ks=(128, 64), vs=(128, 64),
             slots=FAKE):
        ks, vs = ((ctypes.c_int64 * 2)(*x) for x in (ks, vs))
        return lib.iree_mi355x_append_kv_f16(ctypes.byref(c), k, v, rows, ks,
                                             vs, slots, None)

    assert lib.iree_mi355x_append_kv_f16(None, FAKE, FAKE, 3, None, None,
                                         FAKE, None) == pkg.INVALID_ARGUMENT
    for kw in (dict(rows=-1), dict(k=None), dict(v=None), dict(slots=None),
               dict(ks=(-8, 64)), dict(vs=(128, -8))):
        assert call(**kw) == pkg.INVALID_ARGUMENT, kw
    for kw in (dict(k=FAKE + 8), dict(v=FAKE + 2), dict(slots=FAKE + 1),
               dict(ks=(132, 64)), dict(vs=(128, 4))):
        assert call(**kw) == pkg.MISALIGNED, kw
    assert call(rows=1 << 31) == pkg.UNSUPPORTED
    # nothing to do
    assert call(rows=0, k=None, v=None, slots=None) == pkg.OK
    assert call(c=cache(pkg, pages=0, k=None, v=None)) == pkg.OK
    assert call(c=cache(pkg, kv_heads=0)) == pkg.OK


def paged(pkg, c=None, **kw):
    a = pkg.PagedAttentionArgs(
        cache=c or cache(pkg), q=FAKE, o=FAKE, row_starts=FAKE, lengths=FAKE,
        block_table=FAKE, prefix_pages=FAKE, rows=6, heads=8, batch=3,
        table_width=2, table_stride=2, prefix_length=40, scale=0.125)
    a.q_strides[:] = a.o_strides[:] = [512, 64]
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


def attend(pkg, c=None, ws=None, wsb=0, **kw):
    a = paged(pkg, c, **kw)
    return pkg.library().iree_mi355x_shared_prefix_attention_f16(
        ctypes.byref(a), ws, wsb, None)


def test_attention_argument_errors(pkg):
    lib = pkg.library()
    assert lib.iree_mi355x_shared_prefix_attention_f16(
        None, None, 0, None) == pkg.INVALID_ARGUMENT
    for kw in (dict(flags=1), dict(rows=-1), dict(heads=-1), dict(batch=-1),
               dict(table_width=-1), dict(table_stride=-1),
               dict(prefix_length=-1), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(heads=7), dict(q=None),
               dict(o=None), dict(row_starts=None), dict(lengths=None),
               dict(block_table=None), dict(prefix_pages=None),
               dict(table_stride=1), dict(q_strides=[-8, 64]),
               dict(o_strides=[512, 32]), dict(o_strides=[32, 64])):
        assert attend(pkg, **kw) == pkg.INVALID_ARGUMENT, kw
    for kw in (dict(q=FAKE + 8), dict(o=FAKE + 4), dict(lengths=FAKE + 1),
               dict(q_strides=[508, 64]), dict(o_strides=[510, 64]),
               dict(ws=FAKE + 8, wsb=1 << 20)):
        assert attend(pkg, **kw) == pkg.MISALIGNED, kw
    for kw in (dict(rows=1 << 30), dict(batch=1 << 31),
               dict(prefix_length=1 << 30), dict(heads=1 << 17),
               dict(rows=1 << 27, prefix_length=9999, ws=FAKE, wsb=1 << 62)):
        assert attend(pkg, **kw) == pkg.UNSUPPORTED, kw
    # nothing to do
    for kw in (dict(rows=0), dict(heads=0), dict(batch=0)):
        assert attend(pkg, q=None, o=None, **kw) == pkg.OK, kw


def test_attention_workspace(pkg):
    """Parts of rows: 512 workgroups' of 128 rows and both kinds of every
    row, whatever the lengths are."""
    def need(**kw):
        a = paged(pkg, **kw)
        return (pkg.library().
                iree_mi355x_shared_prefix_attention_workspace_bytes(
                    ctypes.byref(a)))

    # f32 rows of the head-dim bucket, their (max, sum), and where they are
    rows = 2 * 6 * 8 + 512 * 128
    full = (256 << 10) + rows * (64 + 2) * 4 + 2 * 6 * 4 * 8
    assert need(prefix_length=8192) == need(table_width=99) == full
    assert need(rows=5000, prefix_length=8192) > full + 2 * 8 * 4994 * 66 * 4
    # up to 1024 keys no row has parts; up to 768 where a request must have
    # more than 16 rows, 512 where there can be more tiles than run at once
    assert need() == need(prefix_length=1024 - 32) == 0
    assert need(prefix_length=1025 - 32) == full
    assert need(rows=50, prefix_length=768 - 32) == 0
    assert need(rows=50, prefix_length=769 - 32) > full
    assert need(rows=50000, prefix_length=512 - 32) == 0
    assert need(rows=50000, prefix_length=513 - 32) > full
    for kw in (dict(rows=0), dict(heads=7), dict(batch=0), dict(rows=1 << 40),
               dict(prefix_length=-1)):
        assert need(**kw) == 0
    assert (pkg.library().iree_mi355x_shared_prefix_attention_workspace_bytes(
        None)) == 0
