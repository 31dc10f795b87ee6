"""Edges of the channels-last operators on the CPU: what the library and the
Python layer refuse and take before anything reaches a device. No compute call
is made here."""
import ctypes as C
import random

import pytest

from simtgo_b200 import _lib

torch = pytest.importorskip("torch")
from simtgo_b200 import channels as ch  # noqa: E402

P = C.c_void_p
MB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture
def calls(monkeypatch):
    """The library calls that the Python layer would make, with CPU or meta
    tensors in the place of CUDA ones."""
    made = []
    monkeypatch.setattr(ch, "_on_gpu", lambda t, name: t.get_device())
    monkeypatch.setattr(ch, "_call", lambda *args: made.append(args))
    return made


def test_extents_past_32_bits_are_refused(calls):
    """None may wrap on its way into the library's 32-bit arguments."""
    def meta(*shape, dtype=torch.float16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    wide = (1 << 32) + 8
    for shape in ((wide,), (1, wide), (3, wide), (1, 1 << 31)):
        x = meta(*shape)
        k = ch.NewCheckpoint(x)
        for call in (lambda: ch.Pack8(k, x), lambda: ch.Unpack8(x, k), lambda: ch.Gated(x, x),
                     lambda: ch.GatedBackward(x, None, x, x)):
            with pytest.raises(_lib.SimtgoError, match="channels") as e:
                call()
            assert e.value.code == _lib.ESIZE
    for shape in ((wide, 2, 8), (2, wide, 8), (2, 1 << 16, 1 << 17, 8), (1, 2, wide)):
        x = meta(*shape)
        m = meta(shape[0], 1, dtype=torch.float32)
        for call in (lambda: ch.GroupNorm(x, x, groups=1),
                     lambda: ch.GroupNormBackward(x, None, None, x, x, m, m, groups=1)):
            with pytest.raises(_lib.SimtgoError) as e:
                call()
            assert e.value.code == _lib.ESIZE
    assert not calls
    ch.Pack8(ch.NewCheckpoint(meta(3, (1 << 31) - 1)), meta(3, (1 << 31) - 1))
    assert len(calls) == 1


def norm_cfg(n=2, s=8, c=16, g=4, **pitch):
    p = {k: v for f in ("x", "y", "d") for k, v in ((f + "_sample", s * c), (f + "_row", c))}
    p.update(pitch)
    return _lib.GroupNormConfig(**p, samples=n, positions=s, channels=c, groups=g, type=0,
                                param_type=0, act=0, block=32, act_param=0.5, eps=1e-5)


def forward(lib, cfg, y, x):
    return lib.simtgo_GroupNorm(P(y), None, None, P(x), None, None, None, None, None, C.byref(cfg),
                                None)


def test_parts_of_one_batch_do_not_overlap(lib):
    E = _lib
    base = 4 * MB

    def both(off, n=3, s=8, sample=320, row=16):
        """x at the start of a buffer, y `off` elements on, the same pitches."""
        return forward(lib, norm_cfg(n=n, s=s, x_sample=sample, x_row=row, y_sample=sample,
                                     y_row=row), base + 4 * off, base)

    # Crops of positions: 0..8 and 8..16, 12..20 of samples of 20 rows.
    for off in (8 * 16, 12 * 16):
        assert both(off) not in (E.EALIAS, E.EARG)
    for off in (7 * 16, 13 * 16, 8 * 16 - 1, 12 * 16 + 1, 0):
        assert both(off) == E.EALIAS
    # Every second sample, every second row, and the rows' other halves.
    assert both(320, sample=640, s=20) not in (E.EALIAS, E.EARG)
    assert both(16, sample=1008, row=48, s=20) not in (E.EALIAS, E.EARG)
    assert both(16 + 16, sample=1008, row=48, s=20) not in (E.EALIAS, E.EARG)
    assert both(17 + 16, sample=1008, row=48, s=20) == E.EALIAS
    # Time-major: a position's samples lie together.
    assert both(5 * 16, n=3, s=8, sample=16, row=160) not in (E.EALIAS, E.EARG)
    assert both(2 * 16, n=3, s=8, sample=16, row=160) == E.EALIAS


def test_overlaps_against_every_element(lib):
    """Random pitches and offsets: an overlap is always refused, and what has no
    overlap is taken where both have the same pitches."""
    rng = random.Random(5)
    free = clash = 0
    for _ in range(3000):
        n, s, c = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 6)
        row = rng.randint(c, 3 * c)
        sample = (s - 1) * row + c + rng.choice((0, 1, row, 3 * row, rng.randint(0, 40)))
        if rng.random() < 0.3:   # time-major
            sample, row = row, (n - 1) * row + c + rng.randint(0, 30)
        off = rng.randint(-120, 120)
        same = rng.random() < 0.7
        ys, yr = (sample, row) if same else (sample + rng.randint(0, 9), row)
        x = {i * sample + j * row + k for i in range(n) for j in range(s) for k in range(c)}
        y = [off + i * ys + j * yr + k for i in range(n) for j in range(s) for k in range(c)]
        if len(set(y)) < len(y):
            continue
        rc = forward(lib, norm_cfg(n=n, s=s, c=c, g=1, x_sample=sample, x_row=row, y_sample=ys,
                                   y_row=yr), 4 * MB + 4 * off, 4 * MB)
        if x & set(y):
            clash += 1
            assert rc == _lib.EALIAS, (n, s, c, sample, row, ys, yr, off)
        elif same:
            free += 1
            assert rc != _lib.EALIAS, (n, s, c, sample, row, off)
    assert free > 300 and clash > 300


def test_layouts_without_elements(calls):
    for shape in ((2, 0, 8), (0, 3, 8), (2, 3, 0), (2, 0, 4, 8), (2, 3, 0, 8), (2, 5, 0)):
        x = torch.zeros(*shape)
        ch._rows(x, "x")
        ch.Gated(x, x)
        ch.Pack8(ch.NewCheckpoint(x, 32), x)
        if shape[-1]:
            ch._batch(x, "x")
            ch.GroupNorm(x, x, groups=2)
    ch._rows(torch.zeros(3, 4, 5, 8)[:, :0, :2], "x")
    ch._batch(torch.zeros(3, 4, 5, 8)[:, :0, :2], "x")
    with pytest.raises(TypeError, match="one pitch"):
        ch._rows(torch.zeros(4, 6, 8)[:, :4], "x")


def test_buffers_without_elements_do_not_overlap(lib):
    for y in (4 * MB, 4 * MB + 4):
        rc = forward(lib, norm_cfg(s=0, y_sample=0, x_sample=0), y, 4 * MB)
        assert rc not in (_lib.EALIAS, _lib.EARG)


def test_options_are_read_at_every_call(calls):
    """A number that the caller changes in place is another number."""
    x = torch.zeros(2, 3, 8)
    threshold, eps = torch.tensor(0.5), torch.tensor(1e-3)
    m = torch.zeros(2, 2)
    seen = []
    for t, e in ((0.5, 1e-3), (0.75, 1e-2)):
        threshold.fill_(t)
        eps.fill_(e)
        ch.GroupNorm(x, x, groups=2, act="softclip", threshold=threshold, eps=eps)
        ch.GroupNormBackward(x, None, None, x, x, m, m, groups=2, act="softclip",
                             threshold=threshold, eps=eps)
        ch.Gated(x, x, act="softclip", threshold=threshold)
        ch.GatedBackward(x, None, x, x, act="softclip", threshold=threshold)
        got, calls[:] = [c[-1]._obj for c in calls], []
        assert [round(c.act_param, 6) for c in got] == [t] * 4
        seen.append([round(c.eps, 6) for c in got[:2]])
    assert seen == [[1e-3] * 2, [1e-2] * 2]
