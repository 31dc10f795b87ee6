"""The channels-last operators (simtgo_b200/channels.py) on the GPU against
their definitions in 64 bits (channels_oracle.py, which derives the bounds)."""
import math

import pytest

torch = pytest.importorskip("torch")
import channels_oracle as O  # noqa: E402
from channels_oracle import assert_within  # noqa: E402
from simtgo_b200 import channels as ch  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
ACTS = ["none", "silu", "gelu", "softclip"]
EPS, T = 1e-5, 0.75
MARK = 77.0   # what untouched elements hold


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def lengths_for(n, s):
    """All, none, one, and something between."""
    return [[s, 0, 1, s // 2, s - 1][i % 5] for i in range(n)]


class Case:
    """Inputs and outputs of a group norm, padded places holding NaN."""

    def __init__(self, n, s, c, g, dtype, kind, ragged=False, affine=True, seed=0, ptype=None):
        r = gen(seed)
        self.n, self.s, self.c, self.g, self.dtype, self.kind = n, s, c, g, dtype, kind
        self.x = (normal(r, n, s, c) * (0.5 + torch.rand(c, device="cuda", generator=r))
                  + 0.5 * normal(r, c)).to(dtype)
        self.dy = normal(r, n, s, c, dtype=dtype)
        self.lens = lengths_for(n, s) if ragged else [s] * n
        self.lengths = None
        if ragged:
            self.lengths = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
            pad = torch.arange(s, device="cuda")[None] >= self.lengths[:, None]
            self.x.masked_fill_(pad[..., None], math.nan)
            self.dy.masked_fill_(pad[..., None], math.nan)
        pt = ptype or dtype
        self.w = (1 + 0.3 * normal(r, c)).to(pt) if affine else None
        self.b = (0.3 * normal(r, c)).to(pt) if affine else None
        self.y = torch.full((n, s, c), MARK, dtype=dtype, device="cuda")
        self.dx = torch.full((n, s, c), MARK, dtype=dtype, device="cuda")
        self.mean = torch.full((n, g), MARK, device="cuda")
        self.rstd = torch.full((n, g), MARK, device="cuda")
        self.dw = torch.full((c,), MARK, device="cuda")
        self.db = torch.full((c,), MARK, device="cuda")

    @property
    def args(self):
        return dict(groups=self.g, eps=EPS, act=self.kind, threshold=T, lengths=self.lengths)

    def forward(self, x=None, y=None, **kw):
        ch.GroupNorm(self.y if y is None else y, self.x if x is None else x, self.w, self.b,
                     mean=self.mean, rstd=self.rstd, **self.args, **kw)
        torch.cuda.synchronize()

    def backward(self, x=None, dx=None, dy=None, dw=True, db=True, **kw):
        ch.GroupNormBackward(self.dx if dx is None else dx, self.dw if dw else None,
                             self.db if db else None, self.dy if dy is None else dy,
                             self.x if x is None else x, self.mean, self.rstd, self.w, self.b,
                             **self.args, **kw)
        torch.cuda.synchronize()

    def clean(self, t):
        return torch.nan_to_num(t, nan=0.0) if self.lengths is not None else t

    def padded(self, t):
        """The elements of t at padded positions."""
        return torch.cat([t[i, self.lens[i]:].reshape(-1) for i in range(self.n)])

    def check_forward(self, y=None):
        y = self.y if y is None else y
        want, mean, rstd, bound = O.group_norm(self.clean(self.x), self.w, self.b, self.g, EPS,
                                               self.kind, T, self.lens)
        size = self.clean(self.x).to(O.F64).abs().amax((1, 2))[:, None]
        assert_within("mean", self.mean, mean, 2.0 ** -24 * (mean.abs() + 8 * size) + 1e-38)
        # The variance's roundings are of its own size: a thread's sums are
        # shifted by a value of theirs; halved by the root.
        assert_within("rstd", self.rstd, rstd, 2.0 ** -24 * 16 * rstd)
        for i in range(self.n):
            assert_within(f"y[{i}]", y[i, :self.lens[i]], want[i, :self.lens[i]],
                          bound[i, :self.lens[i]])
        assert (self.padded(y) == MARK).all()

    def check_backward(self, xv=None, dx=None, dw=True, db=True, have_dx=True):
        xv = self.clean(self.x).to(O.F64) if xv is None else xv
        dx = self.dx if dx is None else dx
        wx, ww, wb, bx, bw, bb = O.group_norm_backward(
            self.clean(self.dy), xv, self.mean, self.rstd, self.w, self.b, self.g, self.kind, T,
            self.lens, self.dtype)
        if have_dx:
            for i in range(self.n):
                assert_within(f"dx[{i}]", dx[i, :self.lens[i]], wx[i, :self.lens[i]],
                              bx[i, :self.lens[i]])
            assert (self.padded(dx) == MARK).all()
        if dw:
            assert_within("dweight", self.dw, ww, bw)
        if db:
            assert_within("dbias", self.db, wb, bb)


# ---- group norm: shapes, types, activations ----------------------------------

SHAPES = [  # samples, positions, channels, groups
    (1, 1, 8, 1),
    (2, 3, 5, 5),        # one channel a group, unaligned rows
    (1, 64, 64, 8),
    (3, 100, 130, 13),   # rows of 260 bytes
    (2, 257, 320, 32),
    (2, 33, 2056, 8),    # more than one tile of units
    (1, 5000, 24, 3),
    (2, 7, 8192, 1),     # the most channels, one group
    (5, 50, 1, 1),
    (300, 1, 64, 4),
    (2, 4100, 96, 96),
    (1, 40000, 16, 2),
    (1, 3, 7001, 7001),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_forward_and_backward(shape, dtype):
    i = SHAPES.index(shape)
    k = Case(*shape, dtype, ACTS[(i + TYPES.index(dtype)) % 4], seed=i)
    k.forward()
    k.check_forward()
    k.backward()
    k.check_backward()


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("affine", [False, True])
def test_activations_and_padding(kind, dtype, affine):
    for shape in ((6, 41, 72, 6), (5, 301, 40, 8)):
        k = Case(*shape, dtype, kind, ragged=True, affine=affine, seed=3)
        k.forward()
        k.check_forward()
        k.backward(dw=affine, db=affine)
        k.check_backward(dw=affine, db=affine)


@pytest.mark.parametrize("ptype", TYPES, ids=str)
def test_parameters_of_their_own_type(ptype):
    k = Case(2, 30, 48, 4, BF16, "silu", ptype=ptype)
    k.forward()
    k.check_forward()
    k.backward()
    k.check_backward()


def test_one_parameter_alone_and_outputs_left_out():
    k = Case(2, 30, 48, 4, F32, "gelu")
    k.b = None
    k.forward()
    k.check_forward()
    k.backward(db=False)
    k.check_backward(db=False)
    assert (k.db == MARK).all()
    dx, k.dx = k.dx, None   # parameters alone
    ch.GroupNormBackward(None, k.dw, k.db, k.dy, k.x, k.mean, k.rstd, k.w, None, **k.args)
    torch.cuda.synchronize()
    k.check_backward(dx=dx, have_dx=False)
    y2 = torch.empty_like(k.y)
    ch.GroupNorm(y2, k.x, k.w, None, **k.args)   # no statistics asked for
    torch.cuda.synchronize()
    assert same_bits(y2, k.y)


# Samples that the shared memory of a cluster does not hold: some rows stay
# there, the others come again from L2, through a ring. And extents at the
# limits of a batch, a tile and a thread's rows.
@pytest.mark.parametrize("shape,dtype", [
    ((40, 8192, 64, 4), F32), ((24, 16384, 128, 8), BF16), ((33, 9000, 80, 8), F16),
    ((70, 4097, 72, 9), BF16), ((3, 2049, 2048, 4), BF16), ((2, 513, 2056, 2), F32),
    ((2000, 3, 16, 2), F32), ((5000, 1, 8, 1), BF16), ((1, 100003, 8, 8), F32)], ids=str)
def test_samples_larger_than_shared_memory(shape, dtype):
    k = Case(*shape, dtype, "silu", ragged=True, seed=21)
    kept = ch.NewCheckpoint(k.x, 64)
    k.forward(ckpt=kept)
    k.check_forward()
    k.backward()
    k.check_backward()
    live = torch.cat([torch.arange(k.s, device="cuda") < v for v in k.lens])
    codes, scales = O.pack(k.clean(k.x).reshape(-1, k.c), 64)
    assert torch.equal(kept.codes.reshape(-1, k.c)[live], codes[live])
    assert torch.equal(kept.scales.reshape(live.numel(), -1)[live], scales[live])
    k.dx.fill_(MARK)
    k.backward(x=kept)
    k.check_backward(xv=O.restore(codes, scales, 64).reshape(k.x.shape))


@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2049, 65543])
def test_gated_lengths_around_whole_units(n):
    g = gen(31)
    a, b, dy = (normal(g, 1, n, dtype=BF16) for _ in range(3))
    y, da, db = (torch.full((1, n + 9), MARK, dtype=BF16, device="cuda") for _ in range(3))
    ch.Gated(y[:, :n], a, b, act="silu")
    ch.GatedBackward(da[:, :n], db[:, :n], dy, a, b, act="silu")
    for got, (want, bound) in zip((y, da, db), gated_bounds(
            a.to(O.F64), b.to(O.F64), dy.to(O.F64), "silu", BF16)):
        assert_within("gated", got[:, :n], want, bound)
        assert (got[:, n:] == MARK).all()


# ---- group norm: layouts ------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("layout", ["slice", "time_major", "crop", "offset", "nchw", "pitch"])
def test_layouts(layout, dtype):
    n, s, c, g = 3, 60, 24, 4
    k = Case(n, s, c, g, dtype, "silu")

    def place(t):
        if layout == "slice":        # channels out of a wider batch, rows interleaved
            buf = torch.full((n, s, 3 * c), MARK, dtype=dtype, device="cuda")
            v = buf[:, :, c:2 * c]
        elif layout == "time_major":
            buf = torch.full((s, n, c), MARK, dtype=dtype, device="cuda")
            v = buf.transpose(0, 1)
        elif layout == "crop":       # positions out of longer samples
            buf = torch.full((n, s + 9, c), MARK, dtype=dtype, device="cuda")
            v = buf[:, 5:5 + s]
        elif layout == "offset":     # one element off any wider boundary
            buf = torch.full((n * s * c + 1,), MARK, dtype=dtype, device="cuda")
            v = buf[1:].view(n, s, c)
        elif layout == "nchw":
            buf = torch.full((n, c, 6, 10), MARK, dtype=dtype, device="cuda").to(
                memory_format=torch.channels_last)
            v = buf.permute(0, 2, 3, 1)
            v.copy_(t.view(n, 6, 10, c))
            return v, buf
        else:                        # rows with a gap that keeps them aligned
            buf = torch.full((n, s, c + 8), MARK, dtype=dtype, device="cuda")
            v = buf[:, :, :c]
        v.copy_(t)
        return v, buf

    x, _ = place(k.x)
    y, ybuf = place(k.y)
    dy, _ = place(k.dy)
    dx, dbuf = place(k.dx)
    k.forward(x=x, y=y)
    k.backward(x=x, dy=dy, dx=dx)
    ref = Case(n, s, c, g, dtype, "silu")
    ref.forward()
    ref.backward()
    for got, want in ((y, ref.y), (dx, ref.dx), (k.dw, ref.dw), (k.db, ref.db), (k.mean, ref.mean)):
        assert same_bits(got.reshape(want.shape), want)
    ref.check_forward()
    ref.check_backward()
    for buf, v in ((ybuf, y), (dbuf, dx)):   # nothing beside the view is written
        v.fill_(MARK)
        assert (buf == MARK).all()


def test_broadcast_inputs():
    k = Case(3, 40, 16, 2, F32, "silu")
    one = k.dy[:1, :1]
    k.dy = one.expand(3, 40, 16).contiguous()
    k.forward()
    k.backward(dy=one.expand(3, 40, 16))
    k.check_backward()
    x1 = k.x[:1]
    y = torch.empty_like(k.y)
    ch.GroupNorm(y, x1.expand(3, 40, 16), k.w, k.b, **k.args)
    torch.cuda.synchronize()
    assert same_bits(y[1], y[0]) and same_bits(y[2], k.y[0])


# ---- group norm: numbers that hurt ------------------------------------------------

@pytest.mark.parametrize("s", [50, 3000, 70000])
def test_mean_far_from_zero_and_first_rows_far_out(s):
    k = Case(2, s, 32, 4, F32, "none")
    k.x += 4096.0
    k.x[0, 0] = 1e6    # every thread's shift, were it shared
    k.x[1, 0, 3] = -3e5
    k.forward()
    k.check_forward()
    k.backward()
    k.check_backward()


def test_constant_input():
    k = Case(2, 333, 40, 5, F32, "none")
    k.x.fill_(3.25)
    k.forward()
    # Every deviation is an exact zero.
    assert (k.mean == 3.25).all()
    assert_within("rstd", k.rstd, torch.full_like(k.rstd, 1 / math.sqrt(EPS)).to(O.F64),
                  torch.full_like(k.rstd, 1e-4).to(O.F64))
    assert torch.equal(k.y, k.b.expand_as(k.y))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("s", [40, 9000])
def test_a_bad_value_stays_in_its_group(bad, s):
    k = Case(2, s, 32, 4, F32, "silu")
    k.x[1, 7, 9] = bad
    k.forward()
    assert torch.isnan(k.y[1, :, 8:16]).all() and torch.isnan(k.rstd[1, 1])
    k.y[1, :, 8:16] = 0
    assert torch.isfinite(k.y).all()
    k.backward()
    assert torch.isnan(k.dx[1, :, 8:16]).all() and torch.isnan(k.dw[8:16]).all()
    k.dx[1, :, 8:16] = 0
    assert torch.isfinite(k.dx).all() and torch.isfinite(k.dw[:8]).all()


def test_lengths_beyond_the_batch_are_clamped():
    k = Case(3, 20, 16, 2, F32, "none")
    k.lengths = torch.tensor([50, -4, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    k.lens = [20, 0, 20]
    k.forward()
    k.check_forward()


def test_empty_extents():
    k = Case(3, 0, 16, 2, F32, "none")
    k.forward()
    assert (k.mean == 0).all()
    assert ((k.rstd - 1 / math.sqrt(EPS)).abs() < 1e-3).all()
    k.backward()
    assert (k.dw == 0).all() and (k.db == 0).all()
    k = Case(0, 5, 16, 2, F32, "none")
    k.forward()
    k.backward()
    assert (k.dw == 0).all() and (k.db == 0).all()


# ---- group norm from a checkpoint -----------------------------------------------

@pytest.mark.parametrize("block", ch.BLOCKS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 65, 320, 32), (3, 40, 50, 5), (1, 700, 8, 2),
                                   (2, 20, 4104, 3), (2, 9000, 64, 4)], ids=str)
def test_checkpoint_in_the_same_pass(shape, dtype, block):
    ragged = shape[0] == 3
    k = Case(*shape, dtype, "silu", ragged=ragged)
    kept = ch.NewCheckpoint(k.x, block)
    kept.codes.fill_(55)
    kept.scales.fill_(MARK)
    k.forward(ckpt=kept)
    k.check_forward()
    c = k.c
    codes, scales = O.pack(k.clean(k.x).reshape(-1, c), block)
    live = torch.cat([torch.arange(k.s, device="cuda") < v for v in k.lens])
    got_c, got_s = kept.codes.reshape(-1, c), kept.scales.reshape(live.numel(), -1)
    assert torch.equal(got_c[live], codes[live]) and torch.equal(got_s[live], scales[live])
    assert (got_c[~live] == 55).all() and (got_s[~live] == MARK).all()
    kept.codes.reshape(-1, c)[~live] = 1
    kept.scales.reshape(live.numel(), -1)[~live] = math.nan
    k.backward(x=kept)
    xv = O.restore(codes, scales, block).reshape(k.x.shape)
    k.check_backward(xv=xv)


# ---- checkpoints -------------------------------------------------------------------

@pytest.mark.parametrize("block", ch.BLOCKS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 8), (7, 333), (64, 256), (5, 2049), (1000, 24),
                                   (3, 9000), (1, 40)], ids=str)
def test_pack_and_unpack(shape, dtype, block):
    x = (normal(gen(1), *shape) * torch.exp(2 * normal(gen(2), shape[0], 1))).to(dtype)
    kept = ch.NewCheckpoint(x, block)
    back = torch.full(shape, MARK, dtype=dtype, device="cuda")
    ch.Pack8(kept, x)
    ch.Unpack8(back, kept)
    codes, scales = O.pack(x, block)
    assert torch.equal(kept.codes, codes) and torch.equal(kept.scales, scales)
    assert torch.equal(back, O.restore(codes, scales, block).float().to(dtype))
    # Half a code step from the input, plus the roundings of the format.
    step = kept.scales.repeat_interleave(block, 1)[:, :shape[1]].to(O.F64)
    assert_within("restored", O.restore(codes, scales, block), x.to(O.F64), step * 0.50002)


def test_pack_edge_values():
    block = 32
    x = torch.zeros(9, 64, device="cuda")
    x[1, :4] = torch.tensor([1e-38, -1e-45, 2e-39, 3e-42])      # below the scale's floor
    x[2, :3] = torch.tensor([3.4e38, -3.4e38, 1.7e38])
    x[3, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -3.5])  # ties, to even
    x[4, 5] = math.nan
    x[5, 6] = math.inf
    x[6, 40] = -math.inf
    x[7] = -2.0
    x[8, 0] = 2.0 ** -100
    kept = ch.NewCheckpoint(x, block)
    back = torch.empty_like(x)
    ch.Pack8(kept, x)
    ch.Unpack8(back, kept)
    codes, scales = O.pack(x, block)
    ok = torch.isfinite(scales).repeat_interleave(block, 1)
    assert torch.equal(kept.codes[ok], codes[ok])
    assert torch.equal(torch.isnan(kept.scales), torch.isnan(scales))
    assert torch.equal(kept.scales[torch.isfinite(scales)], scales[torch.isfinite(scales)])
    assert (back[0] == 0).all() and (back[1] == 0).all()
    assert kept.codes[3, :6].tolist() == [127, 0, 2, 2, 0, -4]
    assert torch.isnan(back[4, :32]).all() and (back[4, 32:] == 0).all()
    assert torch.isnan(back[5, :32]).all() and torch.isnan(back[6, 32:]).all()
    assert (back[7] == -2.0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_pack_strided_rows(dtype):
    wide = normal(gen(4), 37, 300, dtype=dtype)
    for lo, c in ((0, 96), (8, 96), (1, 95), (3, 64)):
        x = wide[:, lo:lo + c]
        kept = ch.NewCheckpoint(x, 32)
        ch.Pack8(kept, x)
        codes, scales = O.pack(x, 32)
        assert torch.equal(kept.codes, codes) and torch.equal(kept.scales, scales)
        out = torch.full((37, 300), MARK, dtype=dtype, device="cuda")
        ch.Unpack8(out[:, lo:lo + c], kept)
        assert torch.equal(out[:, lo:lo + c], O.restore(codes, scales, 32).float().to(dtype))
        out[:, lo:lo + c] = MARK
        assert (out == MARK).all()


def test_pack_three_axes_and_nothing():
    x = normal(gen(5), 3, 4, 40)
    kept = ch.NewCheckpoint(x, 64)
    ch.Pack8(kept, x)
    codes, scales = O.pack(x.reshape(-1, 40), 64)
    assert torch.equal(kept.codes.reshape(-1, 40), codes)
    assert kept.scales.shape == (3, 4, 1) and torch.equal(kept.scales.reshape(-1, 1), scales)
    for shape in ((0, 40), (5, 0)):
        e = torch.empty(*shape, device="cuda")
        k = ch.NewCheckpoint(e, 32)
        ch.Pack8(k, e)
        ch.Unpack8(e, k)
        ch.Gated(e, torch.empty_like(e))


# ---- the gated unit -----------------------------------------------------------------

def gated_bounds(a, b, dy, kind, dtype):
    """y, da, db and bounds. The activation within ev of its value (its
    argument is exact), each product one rounding, then the type's."""
    fast = dtype != F32
    ev = 2.0 ** -19 if fast else 2.0 ** -21
    f, s = O.act(a, kind, T), O.dact(a, kind, T)
    u = O.HALF_STEP[dtype]

    def bound(v, e):
        return u * v.abs() + e + O.TINY[dtype]

    gb = torch.ones_like(a) if b is None else b
    y, da, db = f * gb, dy * gb * s, dy * f
    ef, es = ev * a.abs() + 2.0 ** -23 * f.abs(), 2 * ev * (1 + a.abs())
    return ((y, bound(y, gb.abs() * ef + 2.0 ** -23 * y.abs())),
            (da, bound(da, (dy * gb).abs() * es)),
            (db, bound(db, dy.abs() * ef + 2.0 ** -23 * db.abs())))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 8000), (9, 1111), (700, 72), (3, 2056)], ids=str)
def test_gated(shape, kind, dtype):
    g = gen(7)
    a, b, dy = (2 * normal(g, *shape)).to(dtype), normal(g, *shape, dtype=dtype), normal(
        g, *shape, dtype=dtype)
    y, da, db = (torch.full(shape, MARK, dtype=dtype, device="cuda") for _ in range(3))
    args = dict(act=kind, threshold=T)
    ch.Gated(y, a, b, **args)
    ch.GatedBackward(da, db, dy, a, b, **args)
    for name, got, (want, bound) in zip(("y", "da", "db"), (y, da, db), gated_bounds(
            a.to(O.F64), b.to(O.F64), dy.to(O.F64), kind, dtype)):
        assert_within(name, got, want, bound)
    ch.Gated(y, a, **args)                  # without a gate
    ch.GatedBackward(da, None, dy, a, **args)
    want = gated_bounds(a.to(O.F64), None, dy.to(O.F64), kind, dtype)
    assert_within("act(a)", y, *want[0])
    assert_within("da alone", da, *want[1])
    db2 = torch.empty_like(db)
    ch.GatedBackward(None, db2, dy, a, b, **args)
    assert same_bits(db, db2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("block", ch.BLOCKS)
@pytest.mark.parametrize("shape", [(1, 40), (33, 520), (65, 1111), (4, 4096)], ids=str)
def test_gated_from_checkpoints_in_one_buffer(shape, block, dtype):
    """Both inputs and both gradients as halves of one buffer."""
    r, c = shape
    g = gen(8)
    ab = (1.5 * normal(g, r, 2 * c)).to(dtype)
    a, b = ab[:, :c], ab[:, c:]
    dy = normal(g, r, c, dtype=dtype)
    y = torch.empty(r, c, dtype=dtype, device="cuda")
    dab = torch.full((r, 2 * c), MARK, dtype=dtype, device="cuda")
    ka, kb = ch.NewCheckpoint(a, block), ch.NewCheckpoint(b, block)
    ch.Gated(y, a, b, act="silu", a_ckpt=ka, b_ckpt=kb)
    ch.GatedBackward(dab[:, :c], dab[:, c:], dy, ka, kb, act="silu")
    va, vb = [], []
    for k, t, v in ((ka, a, va), (kb, b, vb)):
        codes, scales = O.pack(t, block)
        assert torch.equal(k.codes, codes) and torch.equal(k.scales, scales)
        v.append(O.restore(codes, scales, block))
    assert_within("y", y, *gated_bounds(a.to(O.F64), b.to(O.F64), dy.to(O.F64), "silu", dtype)[0])
    _, wda, wdb = gated_bounds(va[0], vb[0], dy.to(O.F64), "silu", dtype)
    assert_within("da", dab[:, :c], *wda)
    assert_within("db", dab[:, c:], *wdb)


def test_gated_extreme_inputs():
    for dtype in TYPES:
        big = 6e4 if dtype == F16 else 1e38
        a = torch.tensor([[big, -big, 200.0, -200.0, 88.0, -88.0, 0.0, -0.0]], device="cuda").to(
            dtype)
        one = torch.ones_like(a)
        for kind in ACTS:
            y, da = torch.empty_like(a), torch.empty_like(a)
            ch.Gated(y, a, act=kind, threshold=T)
            ch.GatedBackward(da, None, one, a, act=kind, threshold=T)
            want = O.act(a.to(O.F64), kind, T)
            slope = O.dact(a.to(O.F64), kind, T)
            if dtype != F32:   # exp2 of an argument near 128: 2^-24 * 128 and the unit's
                tol = 2.0 ** -16
            else:
                tol = 2.0 ** -16
            u = O.HALF_STEP[dtype]
            # Far below zero SiLU is of the size of e^z: absolute 2^-120.
            assert_within(kind, y, want, (u + tol) * want.abs() + 2.0 ** -120 + O.TINY[dtype])
            assert_within(kind + "'", da, slope, (u + tol) * slope.abs() + 2.0 ** -100
                          + O.TINY[dtype])


# ---- differences -----------------------------------------------------------------

@pytest.mark.parametrize("kind", ACTS)
def test_group_norm_gradient_against_differences(kind):
    n, s, c, g = 2, 5, 6, 2
    k = Case(n, s, c, g, F32, kind, ragged=True, seed=11)
    k.lens = [5, 3]
    k.lengths = torch.tensor(k.lens, dtype=torch.int32, device="cuda")
    r = gen(12)
    k.x, k.dy = normal(r, n, s, c), normal(r, n, s, c)
    k.forward()
    k.backward()
    h = 1e-5

    def loss(x, w, b):
        y = O.group_norm(x, w, b, g, EPS, kind, T, k.lens)[0]
        return sum((y[i, :v] * k.dy[i, :v].to(O.F64)).sum() for i, v in enumerate(k.lens))

    def against(t, grad, rebuild, live):
        t = t.to(O.F64)
        for i in live:
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            want = float(loss(*rebuild(up)) - loss(*rebuild(down))) / (2 * h)
            # h^2 times a third derivative (rstd^3 of about 10), and float32.
            assert abs(float(grad.reshape(-1)[i]) - want) < 1e-4 * (1 + abs(want)), (i, want)

    x, w, b = k.x.to(O.F64), k.w.to(O.F64), k.b.to(O.F64)
    # Softclip's second derivative jumps at the threshold: differences there
    # are off by h times the jump, far inside the bound.
    live = [(i * s + p) * c + q for i, v in enumerate(k.lens) for p in range(v) for q in range(c)]
    against(x, k.dx, lambda v: (v, w, b), live)
    against(w, k.dw, lambda v: (x, v, b), range(c))
    against(b, k.db, lambda v: (x, w, v), range(c))


# ---- streams, graphs, determinism, far offsets ----------------------------------------

def step(k, kept, ga, out):
    """A block of a training step: norm, gate, and both backward passes."""
    ch.GroupNorm(k.y, k.x, k.w, k.b, mean=k.mean, rstd=k.rstd, ckpt=kept, **k.args)
    ch.Gated(out["h"], k.y, ga, act="gelu", a_ckpt=out["ka"], b_ckpt=out["kb"])
    ch.GatedBackward(out["dn"], out["dg"], k.dy, out["ka"], out["kb"], act="gelu")
    ch.GroupNormBackward(k.dx, k.dw, k.db, out["dn"], kept, k.mean, k.rstd, k.w, k.b, **k.args)


def step_state(seed, dtype=BF16, shape=(3, 130, 96, 8)):
    k = Case(*shape, dtype, "silu", seed=seed)
    ga = normal(gen(seed + 50), *shape[:3], dtype=dtype)
    out = {n: torch.zeros_like(k.x) for n in ("h", "dn", "dg")}
    out["ka"], out["kb"] = ch.NewCheckpoint(k.y, 64), ch.NewCheckpoint(ga, 64)
    return k, ch.NewCheckpoint(k.x, 64), ga, out


def results(st):
    k, kept, ga, out = st
    return [t.clone() for t in (k.y, k.mean, k.rstd, out["h"], out["dn"], out["dg"], k.dx, k.dw,
                                k.db, kept.codes, kept.scales)]


@pytest.mark.parametrize("shape", [(3, 130, 96, 8), (2, 20000, 64, 4)], ids=str)
def test_operators_together(shape):
    st = step_state(1, shape=shape)
    k, kept, ga, out = st
    step(*st)
    torch.cuda.synchronize()
    k.check_forward()
    c = k.c
    cy, sy = O.pack(k.y.reshape(-1, c), 64)
    cg, sg = O.pack(ga.reshape(-1, c), 64)
    va, vb = (O.restore(*v, 64).reshape(k.x.shape) for v in ((cy, sy), (cg, sg)))
    want = gated_bounds(k.y.to(O.F64), ga.to(O.F64), k.dy.to(O.F64), "gelu", BF16)
    assert_within("h", out["h"], *want[0])
    _, wda, wdb = gated_bounds(va, vb, k.dy.to(O.F64), "gelu", BF16)
    assert_within("dn", out["dn"], *wda)
    assert_within("dg", out["dg"], *wdb)
    k.dy = out["dn"]
    k.check_backward(xv=O.restore(*O.pack(k.x.reshape(-1, c), 64), 64).reshape(k.x.shape))


def test_same_bits_again_and_on_another_stream():
    st = step_state(2)
    step(*st)
    first = results(st)
    for t in first:
        assert t.numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (st[0].y, st[0].dx, st[3]["h"], st[0].dw):
            t.zero_()
        step(*st)
    side.synchronize()
    assert all(same_bits(a, b) for a, b in zip(first, results(st)))


@pytest.mark.parametrize("shape", [(3, 130, 96, 8), (2, 20000, 64, 4)], ids=str)
def test_two_captured_graphs_replayed_in_turn(shape):
    states = [step_state(3, shape=shape), step_state(4, shape=shape)]
    want = []
    for st in states:
        step(*st)
        want.append(results(st))
    torch.cuda.synchronize()
    graphs = []
    for st in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(*st)
        graphs.append(g)
    for _ in range(3):
        for st in states:
            st[0].y.zero_(), st[0].dx.zero_(), st[0].dw.zero_(), st[3]["h"].zero_()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        step(*step_state(9, shape=shape))   # an eager step beside them
        torch.cuda.synchronize()
        for st, w in zip(states, want):
            assert all(same_bits(a, b) for a, b in zip(results(st), w))


def test_offsets_past_32_bits():
    far = (1 << 31) + 64
    buf = torch.empty(far + 4096, dtype=BF16, device="cuda")
    k = Case(2, 16, 64, 4, BF16, "silu")
    x = buf.as_strided((2, 16, 64), (far, 64, 1))
    x.copy_(k.x)
    y = torch.empty(far + 4096, dtype=BF16, device="cuda").as_strided((2, 16, 64), (far, 64, 1))
    k.forward(x=x, y=y)
    y2 = k.y
    k.forward()
    assert same_bits(y, y2)
    k.backward(x=x, dx=y)
    k.backward()
    assert same_bits(y, k.dx)
    rows = buf.as_strided((2, 640), (far, 1))
    rows.copy_(normal(gen(1), 2, 640, dtype=BF16))
    kept = ch.NewCheckpoint(rows, 128)
    ch.Pack8(kept, rows)
    codes, scales = O.pack(rows.contiguous(), 128)
    assert torch.equal(kept.codes, codes) and torch.equal(kept.scales, scales)


def test_more_than_2_31_elements():
    r, c = (1 << 20) + 3, 2056   # 2^31 codes and some
    x = torch.empty(r, c, dtype=BF16, device="cuda")
    x.copy_(torch.arange(c, device="cuda", dtype=F32).sub(1000).to(BF16).expand(r, c))
    x[-1] = x[-1].flip(0)
    kept = ch.NewCheckpoint(x, 256)
    back = torch.empty_like(x)
    ch.Pack8(kept, x)
    ch.Unpack8(back, kept)
    for row in (0, r // 2, r - 1):
        codes, scales = O.pack(x[row:row + 1], 256)
        assert torch.equal(kept.codes[row:row + 1], codes)
        assert torch.equal(back[row:row + 1], O.restore(codes, scales, 256).float().to(BF16))


def test_group_norm_of_more_than_2_31_elements():
    """A sample whose rows repeat has the statistics of one period, so its last
    rows have the outputs of the period's."""
    s, c, times = 4096, 136, 4100
    k = Case(1, s, c, 17, BF16, "silu", seed=5)
    k.forward()
    kept = ch.NewCheckpoint(k.x, 64)
    ch.Pack8(kept, k.x)
    x = k.x.repeat(1, times, 1)
    assert x.numel() > 1 << 31
    y = torch.empty_like(x)
    big = ch.NewCheckpoint(x, 64)
    mean, rstd = torch.empty_like(k.mean), torch.empty_like(k.rstd)
    ch.GroupNorm(y, x, k.w, k.b, mean=mean, rstd=rstd, ckpt=big, **k.args)
    assert_within("mean", mean, k.mean.to(O.F64), 1e-6 + 0 * k.mean.to(O.F64))
    assert_within("rstd", rstd, k.rstd.to(O.F64), 1e-5 * k.rstd.to(O.F64))
    for part in (y[:, :s], y[:, -s:]):   # the same z to 1e-5, so at most a step apart
        assert_within("y", part, k.y.to(O.F64), 2.0 ** -7 * k.y.to(O.F64).abs() + 1e-4)
    for part in (slice(None, s), slice(-s, None)):
        assert torch.equal(big.codes[:, part], kept.codes)
        assert torch.equal(big.scales[:, part], kept.scales)


def test_capture_of_shapes_not_run_before():
    """After the device's first call, a graph may hold calls of any shape."""
    warm = Case(1, 8, 8, 1, F32, "none")
    warm.forward()
    warm.backward()
    a, b = Case(3, 77, 56, 7, F16, "gelu", seed=8), Case(1, 30000, 40, 5, F16, "gelu", seed=9)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for k in (a, b):
            ch.GroupNorm(k.y, k.x, k.w, k.b, mean=k.mean, rstd=k.rstd, **k.args)
            ch.GroupNormBackward(k.dx, k.dw, k.db, k.dy, k.x, k.mean, k.rstd, k.w, k.b, **k.args)
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    for k in (a, b):
        k.check_forward()
        k.check_backward()
