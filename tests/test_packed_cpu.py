"""Packed rows without a GPU: what the Python operators and the C-ABI refuse
before anything is launched, and the workspace that attention asks for."""
import ctypes

import pytest
import torch

H, F, I32 = torch.float16, torch.float32, torch.int32
FAKE = 1 << 20


def z(*shape, dtype=H):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape):
    return torch.zeros(*shape, dtype=I32)


# ---------------------------------------------------------------- operators --

def refuses(fn, good):
    def bad(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            fn(**{**good, **kw})
    return bad


def test_rotary_checks(pkg):
    bad = refuses(pkg.rotary, dict(
        q=z(5, 4, 16), k=z(5, 2, 16), positions=i(3, 5),
        frequencies=z(6, dtype=F), sections=(1, 2, 3)))
    bad("3-D f16", TypeError, q=z(5, 64))
    bad("3-D f16", TypeError, q=z(5, 4, 16, dtype=F))
    bad("3-D f16", TypeError, k=z(5, 16, 2).transpose(1, 2))
    bad("k must be", k=z(4, 2, 16))
    bad("k must be", k=z(5, 2, 24))
    bad("positions must be", positions=i(3, 4))
    bad("int32", TypeError, positions=torch.zeros(3, 5, dtype=torch.int64))
    bad("positions must be", positions=i(2, 3, 5))
    bad("unit column", positions=i(5, 3).t())
    bad("float32", TypeError, frequencies=z(6))
    bad("1-D", frequencies=z(2, 3, dtype=F))
    bad("unit column", frequencies=z(12, dtype=F)[::2])
    bad("sections for 3 axes", sections=None)
    bad("sections for 1 axes", positions=i(5))
    bad("1 to 4", positions=i(5, 5), sections=(1, 1, 1, 1, 2))
    bad("must be the 6", sections=(1, 2, 2))
    bad("must be the 6", sections=(-1, 4, 3))
    bad("at most head_dim", frequencies=z(9, dtype=F), sections=(3, 3, 3))
    bad("q_out must be", q_out=z(5, 4, 24))
    bad("k_out must be", k_out=z(5, 4, 16))
    bad("without k", k=None, k_out=z(5, 2, 16))
    bad("device", TypeError)
    bad("device", TypeError, k=None)


def test_rotary_sections_are_integers(pkg):
    """Refused in either order, and a refused call leaves nothing behind that a
    good one of equal sections would be given."""
    def call(sections, n, axes=None):
        positions = i(5) if axes is None else i(axes, 5)
        pkg.rotary(z(5, 4, 2 * n), None, positions, z(n, dtype=F), sections)

    for n in (13, 29):
        with pytest.raises(TypeError, match="sections must be integers"):
            call((float(n),), n)
        for good in ((n,), [n], None, torch.tensor([n])):
            with pytest.raises(TypeError, match="device"):
                call(good, n)
        with pytest.raises(TypeError, match="sections must be integers"):
            call((float(n),), n)
    for bad in ((6.0, 1, 2), ("6", 1, 2), (None,) * 3, 9, torch.ones(3) * 3):
        with pytest.raises(TypeError, match="sections must be integers"):
            call(bad, 9, 3)
    assert all(type(n) is int for n in pkg._sections((13,), 1, 13, 26))


def test_tree_masks_checks(pkg):
    bad = refuses(pkg.tree_masks, dict(parents=i(9), row_starts=i(3),
                                       words=2))
    bad("int32", TypeError, parents=torch.zeros(9, dtype=torch.int64))
    bad("1-D", parents=i(3, 3))
    bad("int32", TypeError, row_starts=None)
    bad("row_starts", row_starts=i(0))
    bad("words", words=0)
    bad("device", TypeError)


def test_tree_attention_checks(pkg):
    bad = refuses(pkg.tree_attention, dict(
        q=z(5, 6, 16), k_cache=z(4, 2, 8, 16), v_cache=z(4, 2, 8, 24),
        row_starts=i(4), lengths=i(3), block_table=i(3, 2), masks=i(5, 1),
        prefix_pages=i(2), prefix_length=16))
    bad("masks must be", masks=i(4, 1))
    bad("masks must be", masks=i(5, 0))
    bad("2-D", masks=i(5))
    bad("unit column", masks=i(2, 5).t())
    bad("int32", TypeError, masks=z(5, 1))
    bad("int32", TypeError, masks=None)
    bad("q must be", q=z(5, 6, 24))
    bad("prefix_pages hold", prefix_length=17)
    bad("o must be", o=z(5, 6, 16))
    bad("device", TypeError)


def test_packed_attention_checks(pkg):
    good = dict(q=z(5, 6, 16), k=z(9, 2, 16), v=z(9, 2, 24), row_starts=i(4),
                key_starts=i(4))
    bad = refuses(pkg.packed_attention, good)
    bad("3-D f16", TypeError, q=z(5, 96))
    bad("3-D f16", TypeError, k=z(9, 2, 16, dtype=F))
    bad("k must be", k=z(9, 2, 24))
    bad("v must be", v=z(8, 2, 24))
    bad("v must be", v=z(9, 3, 24))
    bad("multiple of 2 KV", q=z(5, 5, 16))
    bad("multiple of 0 KV", k=z(9, 0, 16), v=z(9, 0, 24))
    bad("key_starts must be", key_starts=i(3))
    bad("need key_starts", key_starts=None)
    bad("row_starts", row_starts=i(0), key_starts=i(0))
    bad("int32", TypeError, row_starts=torch.zeros(4, dtype=torch.int64))
    bad("o must be", o=z(5, 6, 16))
    bad("o must be", TypeError, o=z(5, 6, 24), out_dtype=F)
    bad("o must be", TypeError, o=[1])
    bad("unit stride", o=z(5, 24, 6).transpose(1, 2))
    bad("float16 or float32", TypeError, out_dtype=torch.bfloat16)
    bad("float16 or float32", TypeError, o=z(5, 6, 24, dtype=torch.float64))
    bad("device", TypeError)
    bad("device", TypeError, o=z(5, 6, 24, dtype=F))


# -------------------------------------------------------------------- C-ABI --

def fill(args, kw):
    for k, v in kw.items():
        if isinstance(v, (list, tuple)):
            getattr(args, k)[:] = v
        else:
            setattr(args, k, v)
    return args


def masks(pkg, **kw):
    a = fill(pkg.TreeMasksArgs(parents=FAKE, row_starts=FAKE, masks=FAKE,
                               depths=FAKE, rows=5, batch=2, words=1), kw)
    return pkg.library().iree_mi355x_tree_masks(ctypes.byref(a), None)


def test_tree_masks_argument_errors(pkg):
    assert pkg.library().iree_mi355x_tree_masks(None, None) == \
        pkg.INVALID_ARGUMENT
    for kw in (dict(rows=-1), dict(batch=-1), dict(words=0), dict(words=-1),
               dict(parents=None), dict(row_starts=None), dict(masks=None),
               dict(depths=None)):
        assert masks(pkg, **kw) == pkg.INVALID_ARGUMENT, kw
        assert "tree_masks" in pkg.last_error()
    for kw in (dict(rows=1 << 30), dict(batch=1 << 24), dict(words=1 << 25)):
        assert masks(pkg, **kw) == pkg.UNSUPPORTED, kw
    for n in ("parents", "row_starts", "masks", "depths"):
        assert masks(pkg, **{n: FAKE + 2}) == pkg.MISALIGNED
    assert masks(pkg, rows=0, parents=None) == pkg.OK


def rotary(pkg, **kw):
    a = fill(pkg.RotaryArgs(
        q=FAKE, k=FAKE, q_out=FAKE, k_out=FAKE, positions=FAKE,
        frequencies=FAKE, rows=5, heads=4, kv_heads=2, head_dim=64, axes=3,
        sections=(8, 12, 12, 0), position_stride=5, q_strides=(256, 64),
        k_strides=(128, 64), q_out_strides=(256, 64),
        k_out_strides=(128, 64)), kw)
    return pkg.library().iree_mi355x_rotary_f16(ctypes.byref(a), None)


def test_rotary_argument_errors(pkg):
    assert pkg.library().iree_mi355x_rotary_f16(None, None) == \
        pkg.INVALID_ARGUMENT
    for kw in (dict(rows=-1), dict(heads=-1), dict(kv_heads=-1),
               dict(head_dim=-1), dict(position_stride=-1), dict(flags=2),
               dict(sections=(8, -1, 12, 0)), dict(sections=(9, 12, 12, 0)),
               dict(q=None), dict(k=None), dict(q_out=None),
               dict(k_out=None), dict(positions=None),
               dict(frequencies=None), dict(q_strides=(-8, 64)),
               dict(k_out_strides=(128, -8)), dict(q_out_strides=(256, 56)),
               dict(k_out_strides=(56, 64))):
        assert rotary(pkg, **kw) == pkg.INVALID_ARGUMENT, kw
        assert "rotary" in pkg.last_error()
    for kw in (dict(axes=0), dict(axes=5), dict(head_dim=258),
               dict(rows=1 << 31), dict(heads=65536), dict(kv_heads=65536),
               dict(sections=(100, 29, 0, 0)),
               dict(sections=(1 << 62, 1 << 62, 1 << 62, 0))):
        assert rotary(pkg, **kw) == pkg.UNSUPPORTED, kw
    for kw in (dict(q=FAKE + 1), dict(k_out=FAKE + 1),
               dict(positions=FAKE + 2), dict(frequencies=FAKE + 1)):
        assert rotary(pkg, **kw) == pkg.MISALIGNED, kw
    assert rotary(pkg, rows=0, q=None) == pkg.OK
    assert rotary(pkg, heads=0, kv_heads=0, q=None) == pkg.OK


def tree(pkg, masks=FAKE, words=2, stride=2, **kw):
    a = pkg.PagedAttentionArgs(
        q=FAKE, o=FAKE, row_starts=FAKE, lengths=FAKE, block_table=FAKE,
        rows=5, heads=4, batch=3, table_width=4, table_stride=4, scale=1.0)
    fill(a.cache, dict(k=FAKE, v=FAKE, pages=4, page_size=16, kv_heads=2,
                       head_dim=64, head_dim_v=64,
                       k_strides=[2048, 1024, 64],
                       v_strides=[2048, 1024, 64]))
    a.q_strides[:] = a.o_strides[:] = [256, 64]
    fill(a, kw)
    return pkg.library().iree_mi355x_tree_attention_f16(
        ctypes.byref(a), masks, words, stride, None, 0, None)


def test_tree_attention_argument_errors(pkg):
    lib = pkg.library()
    assert lib.iree_mi355x_tree_attention_f16(
        None, FAKE, 1, 1, None, 0, None) == pkg.INVALID_ARGUMENT
    for kw in (dict(masks=None), dict(words=0), dict(words=-1),
               dict(stride=1), dict(stride=-1), dict(rows=-1),
               dict(heads=3), dict(q=None), dict(flags=1)):
        assert tree(pkg, **kw) == pkg.INVALID_ARGUMENT, kw
        assert "tree_attention" in pkg.last_error()
    for kw in (dict(words=1 << 25, stride=1 << 25), dict(stride=1 << 31),
               dict(rows=1 << 30)):
        assert tree(pkg, **kw) == pkg.UNSUPPORTED, kw
    assert tree(pkg, masks=FAKE + 2) == pkg.MISALIGNED
    assert tree(pkg, rows=0, masks=None) == pkg.OK


def packed_args(pkg, **kw):
    return fill(pkg.PackedAttentionArgs(
        q=FAKE, k=FAKE, v=FAKE, o=FAKE, row_starts=FAKE, key_starts=FAKE,
        rows=5, key_rows=9, batch=3, heads=4, kv_heads=2, head_dim=64,
        head_dim_v=64, q_strides=(256, 64), k_strides=(128, 64),
        v_strides=(128, 64), o_strides=(256, 64), scale=1.0, flags=1), kw)


def packed(pkg, ws=None, bytes_=0, **kw):
    return pkg.library().iree_mi355x_packed_attention_f16(
        ctypes.byref(packed_args(pkg, **kw)), ws, bytes_, None)


def test_packed_attention_argument_errors(pkg):
    lib = pkg.library()
    assert lib.iree_mi355x_packed_attention_f16(None, None, 0, None) == \
        pkg.INVALID_ARGUMENT
    for kw in (dict(rows=-1), dict(key_rows=-1), dict(batch=-1),
               dict(heads=-1), dict(kv_heads=-1), dict(head_dim=-8),
               dict(head_dim_v=-8), dict(flags=4), dict(heads=3),
               dict(kv_heads=0), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(q=None), dict(k=None),
               dict(v=None), dict(o=None), dict(row_starts=None),
               dict(key_starts=None), dict(q_strides=(-8, 64)),
               dict(v_strides=(128, -8)), dict(o_strides=(56, 64)),
               dict(o_strides=(256, 56))):
        assert packed(pkg, **kw) == pkg.INVALID_ARGUMENT, kw
        assert "packed_attention" in pkg.last_error()
    for kw in (dict(head_dim=60), dict(head_dim_v=264), dict(head_dim=0),
               dict(rows=1 << 30), dict(key_rows=1 << 30),
               dict(batch=1 << 30), dict(heads=65538),
               dict(k_strides=((1 << 24) + 8, 64)),
               dict(v_strides=(1 << 62, 64)),
               # a head's rows over 64 GiB
               dict(key_rows=1 << 20, k_strides=(1 << 15, 64))):
        assert packed(pkg, **kw) == pkg.UNSUPPORTED, kw
    for kw in (dict(q=FAKE + 8), dict(k=FAKE + 8), dict(v=FAKE + 2),
               dict(o=FAKE + 4), dict(o=FAKE + 8, flags=3),
               dict(row_starts=FAKE + 2), dict(key_starts=FAKE + 1),
               dict(q_strides=(252, 64)), dict(k_strides=(128, 60)),
               dict(v_strides=(132, 64)), dict(o_strides=(258, 64)),
               dict(ws=FAKE + 8, bytes_=1 << 30)):
        assert packed(pkg, **kw) == pkg.MISALIGNED, kw
    for kw in (dict(rows=0, q=None), dict(heads=0, kv_heads=0),
               dict(batch=0)):
        assert packed(pkg, **kw) == pkg.OK, kw


def test_packed_attention_of_too_many_tiles(pkg):
    """2^24 (tile, KV head) pairs are more than a launch has."""
    for batch, rows, heads, kv_heads, d in (
            (1 << 20, 1 << 20, 16, 16, 64), (1 << 24, 1, 1, 1, 128),
            (1, 1 << 27, 16, 16, 64), (1, 1 << 27, 64, 16, 128),
            (1 << 20, 1 << 20, 16, 16, 256)):
        assert packed(pkg, batch=batch, rows=rows, key_rows=rows, heads=heads,
                      kv_heads=kv_heads, head_dim=d, head_dim_v=d,
                      o_strides=(heads * d, d)) == \
            pkg.UNSUPPORTED, (batch, rows)
        assert "too large" in pkg.last_error()


def test_packed_workspace(pkg):
    """Only prompts whose tiles are too few to keep the CUs busy, and whose keys
    are many, are split."""
    def need(**kw):
        return pkg.library().iree_mi355x_packed_attention_workspace_bytes(
            ctypes.byref(packed_args(pkg, **kw)))

    assert pkg.library().iree_mi355x_packed_attention_workspace_bytes(
        None) == 0
    assert need(rows=100, key_rows=100, batch=1) == 0
    assert need(rows=1, key_rows=5000, batch=1) > 0
    assert need(rows=2000, key_rows=2000, batch=1) > 0
    assert need(rows=200000, key_rows=200000, batch=1) == 0
    assert need(rows=0) == need(heads=3) == need(head_dim=300) == 0
    for heads, kv_heads in ((32, 8), (8, 2), (16, 16), (3, 1)):
        most = max(need(rows=rows, key_rows=rows + more, batch=1, heads=heads,
                        kv_heads=kv_heads, head_dim=128, head_dim_v=128)
                   for rows in range(1, 40000, 501) for more in (0, 9000))
        assert 0 < most < 256 << 20
