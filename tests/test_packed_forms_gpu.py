"""The forms of packed attention on the GPU: results of 32 bits, and tiles that
are split along their keys, of every head-dim bucket.

The definition in 64 bits is `Packed`'s, and so is the bound of an f16 result.
"""
import pytest
import torch

from test_packed_gpu import Packed

pytestmark = pytest.mark.gpu
H, F, D, I32 = torch.float16, torch.float32, torch.float64, torch.int32
NAN, INF = float("nan"), float("inf")


def parts(pkg, p):
    """The workspace that the call asks for: 0 where tiles are whole."""
    return pkg._packed_workspace_need(
        p.rows, p.k.shape[0], len(p.added), p.heads, p.hk, p.d, p.dv)


class Packed32(Packed):
    """Packed with the bound of an f32 result.

    A weight 2^(s - m) <= 2^4 is held as two f16 operands of 2^11 times it: the
    first is off by 2^-11 of it, the second by 2^-11 of that, or, where either is
    subnormal, 2^-25, which is 2^-36 of the weights' scale: with p the softmax,
    A = sum p |v| + |o| and a largest weight of 1 at least
      2^-22 A + n 2^-36 (max |v| + |o|).
    exp2's last bits are 2^-22 A at most. The 32-bit sums have two products a
    key, and a part, a rescaling and the last quotient a rounding each: (2 n +
    16) 2^-24 A. The scores are off by (d + 8) 2^-24 S, S = max_j scale sum |q
    k_j|, as an f16 result's. All to first order: 2 % more.
    """

    def check(self, got, scale=None):
        scale = self.d ** -0.5 if scale is None else scale
        assert got.dtype is F
        group, worst = self.heads // self.hk, 0.0
        got = got.double()
        for b, (a, m) in enumerate(zip(self.added, self.keys)):
            r0, k0 = self.starts[b], self.key_starts[b]
            mine = got[r0:r0 + a]
            sees = torch.ones(a, m, dtype=torch.bool, device="cuda")
            if self.causal:
                sees = sees.tril(m - a)
            for h in range(self.heads if a and m else 0):
                q = self.q[r0:r0 + a, h].double()
                k = self.k[k0:k0 + m, h // group].double()
                v = self.v[k0:k0 + m, h // group].double()
                s = (q @ k.t() * scale).masked_fill(~sees, -INF)
                p = torch.softmax(s, 1).nan_to_num(0.0)
                r, n = p @ v, sees.sum(1, keepdim=True)
                big = ((q.abs() @ k.abs().t()).masked_fill(~sees, 0.0)
                       .amax(1, keepdim=True) * abs(scale))
                spread = p @ v.abs() + r.abs()
                far = (2 ** -21 * spread
                       + n * 2 ** -36 * (v.abs().amax(0) + r.abs())
                       + (2 * n + 16 + (self.d + 8) * big) * 2 ** -24 * spread)
                off = (mine[:, h] - r).abs()
                assert bool((off <= 1.02 * far).all()), (
                    b, h, float((off / far.clamp(min=1e-30)).max()))
                worst = max(worst, float((off / far.clamp(min=1e-30)).max()))
            if not m:
                assert bool((mine == 0).all())
        assert bool((got[self.starts[-1]:] == 9).all()), "past the last"
        return worst


FORMS = [
    # added, heads, kv heads, d, dv, keys, split
    ([37, 0, 5], 3, 1, 64, 64, None, False),
    ([300, 17], 2, 2, 64, 64, None, False),
    ([70, 130], 6, 1, 96, 96, None, False),
    ([129, 300], 4, 2, 128, 128, None, False),
    ([90, 200], 4, 1, 192, 128, None, False),
    ([1, 2, 3, 1], 4, 1, 192, 128, None, False),
    ([70, 9, 300], 2, 2, 256, 256, None, False),
    ([1, 1, 2], 2, 1, 256, 256, [400, 0, 30], False),
    ([1, 20], 4, 2, 40, 24, [0, 70], False),
    ([20] * 300, 1, 1, 64, 64, None, False),
    # tiles in parts: many rows, joined one at a time, and few, by groups
    ([1500], 2, 2, 64, 64, None, True),
    ([800], 1, 1, 64, 64, None, True),
    ([1500], 2, 2, 96, 96, None, True),
    ([800], 1, 1, 80, 96, None, True),
    ([1500], 2, 2, 128, 128, None, True),
    ([3, 0, 500], 4, 1, 128, 128, [2000, 90, 700], True),
    ([1500], 2, 2, 192, 128, None, True),
    ([800], 1, 1, 192, 128, None, True),
    ([1500], 2, 2, 256, 256, None, True),
    ([0, 1, 200], 2, 2, 200, 232, [900, 1000, 1100], True),
    # narrow tiles alone
    ([1, 2], 4, 1, 192, 128, [3000, 4000], True),
    ([4] * 40, 16, 4, 192, 128, [1500] * 40, True),
    ([1, 2], 4, 1, 256, 256, [3000, 4000], True),
    ([4] * 40, 16, 4, 256, 256, [1500] * 40, True)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", FORMS)
def test_packed_f32_has_its_bits(pkg, dev, shape, causal):
    """A result of 32 bits is as near to the definition as its sums allow, not
    as f16 weights would be."""
    added, heads, hk, d, dv, keys, split = shape
    print(f"f32 {added[:4]} {heads} {hk} {d} {dv} {causal}", flush=True)
    p = Packed32(added, heads, hk, d, dv, keys, causal, pad=3, seed=d)
    assert (parts(pkg, p) > 0) == split
    worst = p.check(p.call(pkg, dtype=F))
    print(f"of the bound: {worst:.3f}", flush=True)


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_packed_small_weights(pkg, dev, rows, d):
    """One key far ahead of 4000 that share the rest: weights of 3e-5, which
    f16 holds with 9 bits; f32 results keep theirs, f16 ones their bound."""
    print(f"small {rows} {d}", flush=True)
    p = Packed32([rows], 2, 1, d, d, [4000], False, seed=d)
    p.q.zero_()
    p.k.zero_()
    p.q[:, :, 0], p.k[1234, :, 0] = 8.0, 10.4 / 8 * d ** 0.5
    p.k[:, :, 1] = torch.linspace(-1, 1, 4000).half().cuda()[:, None]
    p.q[:, 1, 1] = 1.0
    p.v.abs_()
    p.check(p.call(pkg, dtype=F))
    Packed.check(p, p.call(pkg))


def test_packed_f32_views(pkg, dev):
    """Outputs of 32 bits in the columns of a wider buffer, whole and split."""
    for added, d in (([200, 3], 64), ([1500], 96), ([800], 256)):
        p = Packed32(added, 2, 1, d, d)
        for pad, at in ((8, 4), (4, 0)):
            buf = torch.full((p.rows, 2, d + pad), 9.0, device="cuda")
            p.check(p.call(pkg, buf[..., at:at + d]))
            assert bool((buf[..., :at] == 9).all()
                        and (buf[..., at + d:] == 9).all())


# ------------------------------------------------------- tiles in parts, f16 --

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [s for s in FORMS if s[6]] + [
    # more sequences than lanes
    ([3, 0, 1, 9] * 25, 2, 1, 64, 64, [900, 5, 0, 2700] * 25, True),
    ([1] * 200, 1, 1, 128, 128, [3, 1200] * 100, True),
    ([2, 1, 0, 6] * 20, 1, 1, 256, 256, [1500, 0, 9, 1700] * 20, True)])
def test_packed_parts(pkg, dev, shape, causal):
    added, heads, hk, d, dv, keys, _ = shape
    print(f"parts {added[:4]} {heads} {hk} {d} {dv} {causal}", flush=True)
    p = Packed(added, heads, hk, d, dv, keys, causal, pad=3, seed=d + 1)
    assert parts(pkg, p) > 0
    p.check(p.call(pkg))


SPLIT = [
    # added, heads, kv heads, d, dv, keys
    ([1500], 2, 2, 64, 64, None),
    ([1400, 100], 2, 2, 96, 96, None),
    ([1500], 2, 2, 192, 128, None),
    ([1300], 2, 1, 256, 256, None),
    ([300, 200], 4, 1, 128, 128, [1500, 900]),
    ([1, 2], 4, 1, 192, 128, [3000, 1000]),
    ([1, 2], 4, 1, 256, 256, [3000, 1000]),
    ([40, 2], 1, 1, 64, 64, [60000, 200])]  # of many sequences too


@pytest.mark.parametrize("shape", SPLIT)
def test_packed_parts_nan(pkg, dev, shape):
    """A NaN in a query stays in its row and head, one in a key in the rows that
    see it, whatever part it is in."""
    added, heads, hk, d, dv, keys = shape
    print(f"nan {shape}", flush=True)
    group = heads // hk
    for dtype in (H, F):
        p = Packed(added, heads, hk, d, dv, keys, seed=d)
        assert parts(pkg, p) > 0
        p.q.mul_(0.5)
        clean = p.call(pkg, dtype=dtype)
        want = torch.zeros(p.rows, heads, dtype=torch.bool, device="cuda")
        p.q[0, heads - 1] = NAN
        want[0, heads - 1] = True
        # a key in the middle of the last sequence
        a, n = p.added[-1], p.keys[-1]
        j = n // 2
        p.k[p.key_starts[-2] + j, 0] = NAN
        want[p.starts[-2] + max(0, j - (n - a)):, :group] = True
        got = p.call(pkg, dtype=dtype)
        assert torch.equal(got.isnan().all(2), want)
        assert torch.equal(got.isnan().any(2), want)
        assert torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("d,dv", [(64, 64), (96, 96), (128, 128), (192, 128),
                                  (256, 256)])
def test_packed_parts_infinite_scores(pkg, dev, d, dv):
    """Keys of scores -inf have the weight 0, whole parts of them too: the rows
    behind them are those of a sequence that begins there."""
    lead, n = 400, 1500
    p = Packed([n], 2, 2, d, dv, seed=d)
    assert parts(pkg, p) > 0
    p.q.abs_().clamp_(min=0.01)
    p.k[:lead] = -INF
    got = p.call(pkg)
    rest = Packed32([n - lead], 2, 2, d, dv)
    rest.q, rest.k, rest.v = p.q[lead:], p.k[lead:], p.v[lead:]
    Packed.check(rest, got[lead:])
    rest.check(p.call(pkg, dtype=F)[lead:])


def raw(pkg, p, o, workspace, bytes_, starts, key_starts):
    """The C entry on a workspace of the caller's."""
    import ctypes
    a = pkg.PackedAttentionArgs(
        q=p.q.data_ptr(), k=p.k.data_ptr(), v=p.v.data_ptr(), o=o.data_ptr(),
        row_starts=starts.data_ptr(), key_starts=key_starts.data_ptr(),
        rows=p.rows, key_rows=p.k.shape[0], batch=starts.numel() - 1,
        heads=p.heads, kv_heads=p.hk, head_dim=p.d, head_dim_v=p.dv,
        scale=p.d ** -0.5, flags=(pkg.CAUSAL if p.causal else 0)
        | (pkg.ATTENTION_OUT_F32 if o.dtype is F else 0))
    for name, x in zip("qkvo", (p.q, p.k, p.v, o)):
        getattr(a, name + "_strides")[:] = x.stride()[:2]
    return pkg.library().iree_mi355x_packed_attention_f16(
        ctypes.byref(a), workspace, bytes_,
        torch.cuda.current_stream().cuda_stream)


TOP = 2 ** 31 - 1
BAD = [
    # row and key starts, as shares of the rows and of the keys, or as they are
    ([0, 1.0, 0.3, 1.0], [0, 0.7, 0.3, 1.0]),
    ([-7, 0.5, TOP], [-TOP - 1, 0.4, TOP]),
    ([1.0, 0, 1.0], [1.0, 0, 0.6]),
    ([0, 1.0, 0, 1.0, 0, 1.0], [0, 1.0, 0, 1.0, 0, 1.0]),
    ([0.5, 0.6, 0.9], [0.9, 0.1, 1.0]),
    ([0, 0, 0, 1.0], [TOP, TOP, -1, TOP])]


@pytest.mark.parametrize("shape", SPLIT)
def test_packed_parts_bad_starts(pkg, dev, shape):
    """Starts that do not ascend or lie outside the rows, in the split form: rows
    hold anything, but nothing beside the output or the workspace is written,
    whatever the workspace held, and the next call is right."""
    added, heads, hk, d, dv, keys = shape
    print(f"bad starts {shape}", flush=True)

    def ints(x):
        return torch.tensor(x, dtype=I32, device="cuda")

    for causal, dtype in ((True, H), (False, F)):
        p = Packed(added, heads, hk, d, dv, keys, causal, seed=d)
        n, guard = p.k.shape[0], 4096
        for rows, key_rows in BAD + [([0, 1.0] * 33, [0, 1.0] * 33),
                                     ([1.0, 0] * 40, [0, 1.0] * 40)]:
            starts, key_starts = (
                ints([int(x * t) if isinstance(x, float) else x for x in s])
                for s, t in ((rows, p.rows), (key_rows, n)))
            need = pkg._packed_workspace_need(
                p.rows, n, len(rows) - 1, heads, hk, d, dv)
            if len(rows) <= 4 or n > 60000:
                assert need > 0
            for fill in (0, -1, 0x7f):
                buf = torch.full((p.rows + 2, heads, dv), 9.0, dtype=dtype,
                                 device="cuda")
                ws = torch.full((need + 2 * guard,), fill, dtype=torch.int8,
                                device="cuda")
                ws[:guard] = ws[guard + need:] = 0x5a
                assert raw(pkg, p, buf[1:-1], ws.data_ptr() + guard, need,
                           starts, key_starts) == pkg.OK
                torch.cuda.synchronize()
                assert bool((buf[0] == 9).all() and (buf[-1] == 9).all())
                assert bool((ws[:guard] == 0x5a).all()
                            and (ws[guard + need:] == 0x5a).all())
        # the same workspace, right starts
        buf = torch.full((p.rows, heads, dv), 9.0, dtype=dtype, device="cuda")
        need = parts(pkg, p)
        ws = torch.full((need,), 0x7f, dtype=torch.int8, device="cuda")
        assert raw(pkg, p, buf, ws.data_ptr(), need, ints(p.starts),
                   ints(p.key_starts)) == pkg.OK
        p.check(buf)


def test_packed_f32_captured(pkg, dev):
    """Whole and split calls of 32 bits in a graph, replayed with other lengths
    beside f16 calls on the stream's own workspace."""
    calls = [Packed32([1500], 2, 2, 96, 96, pad=4, seed=1),
             Packed32([200, 90], 2, 1, 64, 64, seed=2)]
    assert [parts(pkg, p) > 0 for p in calls] == [True, False]
    starts = [torch.tensor(p.starts, dtype=I32, device="cuda") for p in calls]
    outs = [torch.full((p.rows, p.heads, p.dv), 9.0, device="cuda")
            for p in calls]
    for p in calls:
        p.k[p.starts[-1]:] = p.v[p.starts[-1]:] = 1.0

    def step():
        for p, s, o in zip(calls, starts, outs):
            pkg.packed_attention(p.q, p.k, p.v, s, o=o)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for first, second in (([1500], [200, 90]), ([1504], [290, 0]),
                          ([700], [1, 280])):
        for p, s, o, added in zip(calls, starts, outs, (first, second)):
            p.added = p.keys = added
            p.starts = p.key_starts = [sum(added[:b])
                                       for b in range(len(added) + 1)]
            s.copy_(torch.tensor(p.starts, dtype=I32))
            o.fill_(9.0)
        graph.replay()
        half = [p.call(pkg) for p in calls]
        torch.cuda.synchronize()
        for p, o, h in zip(calls, outs, half):
            p.check(o)
            Packed.check(p, h)
