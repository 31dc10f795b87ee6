"""Edges of the channels-last operators on the CPU: what the library and the
Python layer refuse and take before anything reaches a device. No compute call
is made here."""
import ctypes as C

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
