"""The channels-last operators on the CPU: what the library and the Python
layer refuse before anything reaches a device, and the formulas the GPU tests
compare with, against each other. No compute call is made here."""
import ctypes as C
import pathlib
import re

import pytest

from simtgo_b200 import _lib

torch = pytest.importorskip("torch")
import channels_oracle as O  # noqa: E402
from simtgo_b200 import channels as ch  # noqa: E402

ROOT = pathlib.Path(__file__).resolve().parent.parent
P = C.c_void_p
MB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def err(lib):
    return lib.simtgo_last_error().decode()


def norm_cfg(n=2, s=8, c=16, g=4, type=0, ptype=0, act=0, block=32, param=0.5, eps=1e-5, **pitch):
    p = {k: v for f in ("x", "y", "d") for k, v in ((f + "_sample", s * c), (f + "_row", c))}
    p.update(pitch)
    return _lib.GroupNormConfig(**p, samples=n, positions=s, channels=c, groups=g, type=type,
                                param_type=ptype, act=act, block=block, act_param=param, eps=eps)


def forward(lib, cfg, y=1 * MB, mean=2 * MB, rstd=3 * MB, x=4 * MB, w=5 * MB, b=6 * MB, ln=None,
            codes=None, scales=None):
    return lib.simtgo_GroupNorm(P(y), P(mean), P(rstd), P(x), P(w), P(b), P(ln), P(codes),
                                P(scales), C.byref(cfg) if cfg else None, None)


def backward(lib, cfg, dx=1 * MB, dw=2 * MB, db=3 * MB, dy=4 * MB, x=5 * MB, codes=None,
             scales=None, mean=6 * MB, rstd=7 * MB, w=8 * MB, b=9 * MB, ln=None):
    return lib.simtgo_GroupNorm_backward(P(dx), P(dw), P(db), P(dy), P(x), P(codes), P(scales),
                                         P(mean), P(rstd), P(w), P(b), P(ln),
                                         C.byref(cfg) if cfg else None, None)


def test_group_norm_refusals(lib):
    E = _lib
    for call in (forward, backward):
        assert call(lib, None) == E.ENULL
        assert call(lib, norm_cfg(n=-1)) == E.EARG
        assert call(lib, norm_cfg(g=5)) == E.EARG and "whole number" in err(lib)
        assert call(lib, norm_cfg(g=0)) == E.EARG
        assert call(lib, norm_cfg(type=3)) == E.EARG
        assert call(lib, norm_cfg(ptype=-1)) == E.EARG
        assert call(lib, norm_cfg(act=4)) == E.EARG
        assert call(lib, norm_cfg(act=3, param=-1.0)) == E.EARG
        assert call(lib, norm_cfg(act=3, param=float("nan"))) == E.EARG
        for eps in (0.0, -1.0, float("nan"), float("inf")):
            assert call(lib, norm_cfg(eps=eps)) == E.EARG and "eps" in err(lib)
        assert call(lib, norm_cfg(c=8200, g=1)) == E.ESIZE
        assert call(lib, norm_cfg(s=(1 << 30) + 1)) == E.ESIZE
        assert call(lib, norm_cfg(n=1 << 20, s=1 << 20, c=8192)) == E.ESIZE
        assert call(lib, norm_cfg(), w=5 * MB + 1) == E.EARG and "aligned" in err(lib)
        assert call(lib, norm_cfg(), ln=10 * MB + 2) == E.EARG
        assert call(lib, norm_cfg(x_row=-16)) == E.EARG and "pitches" in err(lib)
        assert call(lib, norm_cfg(y_sample=1 << 60)) == E.EARG
    assert forward(lib, norm_cfg(), y=None) == E.ENULL
    assert forward(lib, norm_cfg(), x=None) == E.ENULL
    assert forward(lib, norm_cfg(), x=4 * MB + 2) == E.EARG
    assert forward(lib, norm_cfg(), codes=7 * MB) == E.ENULL
    assert forward(lib, norm_cfg(block=48), codes=7 * MB, scales=8 * MB) == E.EARG
    assert forward(lib, norm_cfg(), codes=7 * MB, scales=8 * MB + 2) == E.EARG
    assert backward(lib, norm_cfg(), dy=None) == E.ENULL
    assert backward(lib, norm_cfg(), mean=None) == E.ENULL
    assert backward(lib, norm_cfg(), x=None) == E.EARG and "exactly one" in err(lib)
    assert backward(lib, norm_cfg(), codes=10 * MB, scales=11 * MB) == E.EARG
    assert backward(lib, norm_cfg(), x=None, codes=10 * MB) == E.ENULL


def test_group_norm_overlaps(lib):
    E = _lib
    # In place, a statistic inside y, an output inside an input.
    assert forward(lib, norm_cfg(), y=4 * MB) == E.EALIAS
    assert forward(lib, norm_cfg(), mean=1 * MB + 64) == E.EALIAS and "mean" in err(lib)
    assert forward(lib, norm_cfg(), rstd=2 * MB + 16) == E.EALIAS
    assert forward(lib, norm_cfg(), codes=4 * MB + 100, scales=8 * MB) == E.EALIAS
    assert backward(lib, norm_cfg(), dx=4 * MB + 4) == E.EALIAS
    assert backward(lib, norm_cfg(), dw=3 * MB - 32) == E.EALIAS
    # Written rows on top of one another.
    assert forward(lib, norm_cfg(y_row=8)) == E.EALIAS and "rows of y" in err(lib)
    assert forward(lib, norm_cfg(y_sample=0)) == E.EALIAS
    assert backward(lib, norm_cfg(d_row=0)) == E.EALIAS
    # Channel slices of one batch interleave without overlapping.
    wide = dict(x_row=40, x_sample=320, y_row=40, y_sample=320)
    rc = forward(lib, norm_cfg(**wide), y=4 * MB + 64)
    assert rc not in (E.EALIAS, E.EARG)
    assert forward(lib, norm_cfg(**wide), y=4 * MB + 60) == E.EALIAS
    assert forward(lib, norm_cfg(**wide), y=4 * MB + 100) == E.EALIAS
    # Time-major rows, and inputs that share memory.
    rc = forward(lib, norm_cfg(x_row=32, x_sample=16, y_row=32, y_sample=16), w=4 * MB, b=4 * MB)
    assert rc not in (E.EALIAS, E.EARG)
    # Reading one row for every position is no overlap.
    assert forward(lib, norm_cfg(x_row=0, x_sample=0)) not in (E.EALIAS, E.EARG)


def test_empty_group_norm_is_a_no_op(lib):
    assert forward(lib, norm_cfg(n=0), y=None, x=None) == 0
    assert forward(lib, norm_cfg(c=0, g=1), y=None, x=None) == 0
    assert backward(lib, norm_cfg(), dx=None, dw=None, db=None) == 0


def test_checkpoint_refusals(lib):
    E = _lib

    def pack(codes=1 * MB, scales=2 * MB, x=3 * MB, type=0, rows=4, c=100, pitch=100, block=32,
             fn=None):
        if fn is None:
            return lib.simtgo_Pack8(P(codes), P(scales), P(x), type, rows, c, pitch, block, None)
        return lib.simtgo_Unpack8(P(x), P(codes), P(scales), type, rows, c, pitch, block, None)

    for fn in (None, "unpack"):
        for block in (0, -32, 16, 48, 512):
            assert pack(block=block, fn=fn) == E.EARG and "block" in err(lib)
        assert pack(type=7, fn=fn) == E.EARG
        assert pack(rows=-1, fn=fn) == E.EARG and pack(c=-1, fn=fn) == E.EARG
        assert pack(rows=1 << 40, c=1 << 20, fn=fn) == E.ESIZE
        assert pack(codes=None, fn=fn) == E.ENULL and pack(scales=None, fn=fn) == E.ENULL
        assert pack(x=None, fn=fn) == E.ENULL
        assert pack(x=3 * MB + 2, fn=fn) == E.EARG and pack(scales=2 * MB + 1, fn=fn) == E.EARG
        assert pack(pitch=-100, fn=fn) == E.EARG and pack(pitch=1 << 60, fn=fn) == E.EARG
        assert pack(codes=3 * MB + 8, fn=fn) == E.EALIAS
        assert pack(rows=0, codes=None, scales=None, x=None, fn=fn) == 0
        assert pack(c=0, fn=fn) == 0
    assert pack(pitch=99, fn="unpack") == E.EALIAS
    assert pack(pitch=0) not in (E.EARG, E.EALIAS)   # one row packed for every row
    assert pack(scales=1 * MB + 100) == E.EALIAS


def gated_cfg(rows=4, c=40, type=0, act=1, block=32, param=0.5, **pitch):
    p = {k: c for k in ("a_pitch", "b_pitch", "y_pitch", "da_pitch", "db_pitch")}
    p.update(pitch)
    return _lib.GatedUnitConfig(rows=rows, channels=c, type=type, act=act, block=block,
                                act_param=param, **p)


def test_gated_refusals(lib):
    E = _lib

    def fwd(cfg, y=1 * MB, a=2 * MB, b=3 * MB, ac=None, asc=None, bc=None, bsc=None):
        return lib.simtgo_Gated(P(y), P(a), P(b), P(ac), P(asc), P(bc), P(bsc),
                                C.byref(cfg) if cfg else None, None)

    def bwd(cfg, da=1 * MB, db=2 * MB, dy=3 * MB, a=4 * MB, b=5 * MB, ac=None, asc=None, bc=None,
            bsc=None):
        return lib.simtgo_Gated_backward(P(da), P(db), P(dy), P(a), P(b), P(ac), P(asc), P(bc),
                                         P(bsc), C.byref(cfg) if cfg else None, None)

    for call in (fwd, bwd):
        assert call(None) == E.ENULL
        assert call(gated_cfg(rows=-1)) == E.EARG
        assert call(gated_cfg(type=9)) == E.EARG
        assert call(gated_cfg(act=-1)) == E.EARG
        assert call(gated_cfg(act=3, param=float("inf"))) == E.EARG
        assert call(gated_cfg(rows=1 << 45)) == E.ESIZE
        assert call(gated_cfg(rows=0), a=None) == 0
    assert fwd(gated_cfg(), y=None) == E.ENULL and fwd(gated_cfg(), a=None) == E.ENULL
    assert fwd(gated_cfg(), y=2 * MB) == E.EALIAS
    assert fwd(gated_cfg(y_pitch=20)) == E.EALIAS
    assert fwd(gated_cfg(), ac=4 * MB) == E.ENULL
    assert fwd(gated_cfg(block=33), ac=4 * MB, asc=5 * MB) == E.EARG
    assert fwd(gated_cfg(), b=None, bc=4 * MB, bsc=5 * MB) == E.EARG
    assert fwd(gated_cfg(), ac=4 * MB, asc=5 * MB, bc=4 * MB + 80, bsc=6 * MB) == E.EALIAS
    assert bwd(gated_cfg(), a=None) == E.EARG
    assert bwd(gated_cfg(), ac=6 * MB, asc=7 * MB) == E.EARG
    assert bwd(gated_cfg(), bc=6 * MB, bsc=7 * MB) == E.EARG
    assert bwd(gated_cfg(), a=None, ac=6 * MB, asc=7 * MB) == E.EARG   # b is a tensor
    assert bwd(gated_cfg(), b=None) == E.EARG and "db" in err(lib)
    assert bwd(gated_cfg(), da=3 * MB) == E.EALIAS
    # Halves of one buffer, read or written, do not overlap; shifted ones do.
    two = dict(da_pitch=80, db_pitch=80)
    assert bwd(gated_cfg(**two), db=1 * MB + 160) not in (E.EALIAS, E.EARG)
    assert bwd(gated_cfg(**two), db=1 * MB + 156) == E.EALIAS


def test_python_layer_refusals():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(TypeError, match="CUDA"):
        ch.GroupNorm(x, x, groups=2)
    with pytest.raises(TypeError, match="CUDA"):
        ch.Pack8(ch.NewCheckpoint(x), x)
    with pytest.raises(TypeError, match="CUDA"):
        ch.Gated(x, x, x)
    with pytest.raises(ValueError, match="block"):
        ch.NewCheckpoint(x, 100)
    with pytest.raises(TypeError, match="stride 1"):
        ch._batch(x.transpose(1, 2), "x")
    with pytest.raises(TypeError, match="one axis"):
        ch._batch(torch.zeros(2, 4, 6, 8)[:, :, :4], "x")
    with pytest.raises(TypeError, match="one pitch"):
        ch._rows(torch.zeros(4, 6, 8)[:, :4], "x")
    with pytest.raises(ValueError, match="activation"):
        ch._act("relu")
    with pytest.raises(ValueError, match="groups"):
        ch._norm_args(x, 3, None, None, None, None, None)
    with pytest.raises(_lib.LengthError, match="weight"):
        ch._norm_args(x, 2, torch.zeros(9), None, None, None, None)
    with pytest.raises(TypeError, match="float64"):
        ch._type(x.double(), "x")
    with pytest.raises(TypeError):
        ch._batch(torch.zeros(()), "x")


def test_layouts_of_the_python_layer():
    x = torch.zeros(2, 6, 8)
    assert ch._batch(x, "x") == (48, 8)
    assert ch._batch(x.transpose(0, 1), "x") == (8, 48)
    assert ch._batch(torch.zeros(2, 8, 3, 5).to(memory_format=torch.channels_last).permute(
        0, 2, 3, 1), "x") == (120, 8)
    assert ch._rows(torch.zeros(4, 5, 8), "x") == 8
    assert ch._rows(torch.zeros(4, 5, 8)[..., :3], "x") == 8
    assert ch._rows(torch.zeros(4, 1, 8)[:2], "x") == 8
    assert ch._rows(torch.zeros(7), "x") == 7
    assert ch._rows(torch.zeros(1, 1, 7), "x") == 7
    k = ch.NewCheckpoint(torch.zeros(3, 2, 200), 64)
    assert k.codes.shape == (3, 2, 200) and k.scales.shape == (3, 2, 4)


def test_config_layouts_match_the_header_and_the_go_binding():
    head = (ROOT / "include" / "simtgo_b200.h").read_text()
    go = (ROOT / "go" / "b200" / "b200.go").read_text()
    width = {"int64_t": 8, "int32_t": 4, "float": 4, "int64": 8, "int32": 4, "float32": 4}
    for name, struct, gname in (("simtgo_group_norm", _lib.GroupNormConfig, "GroupNormConfig"),
                                ("simtgo_gated_unit", _lib.GatedUnitConfig, "GatedUnitConfig")):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, head, flags=re.S).group(1)
        fields = []
        for decl in body.split(";"):
            if decl.strip():
                ty, names = decl.strip().split(None, 1)
                fields += [(n.strip(), width[ty]) for n in names.split(",")]
        assert fields == [(n, C.sizeof(t)) for n, t in struct._fields_]
        assert C.sizeof(struct) == sum(w for _, w in fields)   # no padding
        gobody = re.search(r"type %s struct \{(.*?)\}" % gname, go, flags=re.S).group(1)
        got = [line.split() for line in gobody.strip().splitlines()]
        assert [width[t] for _, t in got] == [w for _, w in fields]
        assert [n.lower() for n, _ in got] == [n.replace("_", "") for n, _ in fields]


# ---- the formulas against one another ----------------------------------------------

@pytest.mark.parametrize("kind", ["none", "silu", "gelu", "softclip"])
def test_slopes_are_the_activations_differences(kind):
    z = torch.linspace(-6, 6, 997, dtype=O.F64)
    h = 1e-6
    want = (O.act(z + h, kind, 0.7) - O.act(z - h, kind, 0.7)) / (2 * h)
    assert (want - O.dact(z, kind, 0.7)).abs().max() < 1e-6
    assert O.dact(z, kind, 0.7).abs().max() <= O.SLOPE
    second = (O.dact(z + h, kind, 0.7) - O.dact(z - h, kind, 0.7)) / (2 * h)
    assert second.abs().max() <= O.CURVE + 1e-3


@pytest.mark.parametrize("kind", ["none", "silu", "gelu", "softclip"])
def test_oracle_gradient_against_autograd(kind):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 7, 12, generator=g, dtype=O.F64, requires_grad=True)
    w = torch.randn(12, generator=g, dtype=O.F64, requires_grad=True)
    b = torch.randn(12, generator=g, dtype=O.F64, requires_grad=True)
    dy = torch.randn(2, 7, 12, generator=g, dtype=O.F64)
    v = x.reshape(2, 7, 3, 4)
    mean = v.mean((1, 3), keepdim=True)
    rstd = (v.var((1, 3), keepdim=True, unbiased=False) + 1e-5) ** -0.5
    y = O.act(((v - mean) * rstd).reshape(2, 7, 12) * w + b, kind, 0.7)
    (y * dy).sum().backward()
    got = O.group_norm_backward(dy, x.detach(), mean.detach().reshape(2, 3),
                                rstd.detach().reshape(2, 3), w.detach(), b.detach(), 3, kind, 0.7,
                                [7, 7], torch.float32)
    for a, t in zip(got, (x.grad, w.grad, b.grad)):
        assert (a - t).abs().max() < 1e-10


def test_oracle_pack_restores_within_half_a_step():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 100, generator=g)
    codes, scales = O.pack(x, 32)
    assert codes.abs().max() <= 127
    back = O.restore(codes, scales, 32)
    step = scales.repeat_interleave(32, 1)[:, :100].double()
    assert ((back - x.double()).abs() <= 0.50002 * step).all()
