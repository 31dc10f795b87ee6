"""Edges of the channels-last operators on the GPU: launches near a default
limit, outlying first values, far tails, the largest extents and numbers,
other streams, and captures that come first."""
import ctypes as C
import math
import pathlib
import subprocess
import sys
import textwrap

import pytest

torch = pytest.importorskip("torch")
import channels_oracle as O  # noqa: E402
from channels_oracle import assert_within  # noqa: E402
from simtgo_b200 import channels as ch  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5
HERE = pathlib.Path(__file__).resolve().parent


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def fresh_process(code):
    """Runs code where the library has made no call yet."""
    head = f"import sys; sys.path[:0] = [{str(HERE)!r}, {str(HERE.parent)!r}]\n"
    r = subprocess.run([sys.executable, "-c", head + textwrap.dedent(code)], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


def test_first_calls_whose_shared_memory_is_just_under_the_default():
    """A block of the sums over chunks has static shared memory beside the
    dynamic: 1360 channels in groups that are no whole units take 49136 bytes
    and 32. Every access width, before any call that needs more."""
    fresh_process("""
        import torch, channels_oracle as O
        from channels_oracle import assert_within
        from simtgo_b200 import channels as ch
        s = 12000
        for c, groups in ((1360, 16), (2720, 32)):
            for dtype, off in ((torch.float32, 0), (torch.bfloat16, 0), (torch.float16, 0),
                               (torch.float32, 1), (torch.bfloat16, 1), (torch.float16, 1),
                               (torch.bfloat16, 2), (torch.float16, 2)):
                g = torch.Generator(device="cuda").manual_seed(c + off)
                buf = torch.randn(s * c + off, device="cuda", generator=g).to(dtype)
                x = buf[off:].view(1, s, c)
                y = torch.empty_like(buf)[off:].view(1, s, c)
                mean, rstd = torch.empty(2, 1, groups, device="cuda")
                ch.GroupNorm(y, x, groups=groups, mean=mean, rstd=rstd)
                want, m, r, bound = O.group_norm(x, None, None, groups, 1e-5, "none", 1.0, [s])
                assert_within("rstd", rstd, r, 2.0 ** -24 * 16 * r)
                assert_within("y", y, want, bound)
        """)


# Cells (units of eight channels, or single channels) of many rows whose first
# values lie far out: by a sample's single value, by its first row, and by the
# first rows of every stretch of rows that a block may start at.
@pytest.mark.parametrize("where", ["value", "row", "click", "every"])
@pytest.mark.parametrize("shape,far", [
    ((1, 65536, 1024, 16), 4096.0),    # over chunks, groups of whole units
    ((1, 65536, 1900, 38), 4096.0),    # over chunks, other groups
    ((37, 1024, 2048, 1), 3e5),        # clusters
    ((37, 1024, 2040, 2), 3e5)], ids=str)
def test_outlying_first_values(shape, far, where):
    n, s, c, groups = shape
    d = c // groups
    x = normal(gen(41), *shape[:3])
    if where == "value":
        x[:, 0, ::d] = far
    elif where == "row":
        x[:, 0] = far
    elif where == "click":
        x[:, :11, ::d] = -far
    else:
        x[:, ::s // 512, ::8] += far
    y = torch.empty_like(x)
    mean, rstd = torch.empty(2, n, groups, device="cuda")
    ch.GroupNorm(y, x, groups=groups, mean=mean, rstd=rstd)
    step = 8   # the oracle's sums, a few samples at a time
    for lo in range(0, n, step):
        part = x[lo:lo + step]
        wm, wr = O.statistics(part, groups, EPS, [s] * part.shape[0])
        size = part.to(O.F64).abs().amax((1, 2))[:, None]
        # A run of rows is at most three times as long as what came before it,
        # so its squares are at most four times what it adds to the sum of
        # squared deviations; 4 * 8 roundings, halved by the root.
        assert_within("mean", mean[lo:lo + step], wm, 2.0 ** -24 * (wm.abs() + 8 * size))
        assert_within("rstd", rstd[lo:lo + step], wr, 2.0 ** -24 * 16 * wr)


def test_one_row_of_the_most_channels():
    c = (1 << 31) - 1
    x = torch.empty(1, c, dtype=F16, device="cuda")
    x.view(-1)[: 1 << 20].copy_(normal(gen(51), 1 << 20, dtype=F16))
    for lo in range(1 << 20, c, 1 << 28):
        x[0, lo:lo + (1 << 28)] = 0.5
    x[0, -1000:] = normal(gen(52), 1000, dtype=F16)
    kept = ch.NewCheckpoint(x, 32)
    back = torch.empty_like(x)
    ch.Pack8(kept, x)
    ch.Unpack8(back, kept)
    for part in (slice(0, 1 << 20), slice((c - 4096) // 32 * 32, c)):
        codes, scales = O.pack(x[:, part], 32)
        assert torch.equal(kept.codes[:, part], codes)
        first = part.start // 32
        assert torch.equal(kept.scales[:, first:first + scales.shape[1]], scales)
        assert torch.equal(back[:, part], O.restore(codes, scales, 32).float().to(F16))
    ch.Gated(back, x, act="none")
    assert torch.equal(back, x)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_gelu_in_its_negative_tail(dtype):
    """Held to a relative bound: Phi's fit is within 6e-6, exp2's argument of
    at most 104 carries two roundings (9e-6), the rest a few 2^-23; float32: the
    argument of erfc carries two roundings, which it multiplies by z^2 + 1, and
    erfc and the products a few more."""
    z = -torch.linspace(3, 12, 4001, device="cuda", dtype=O.F64).to(dtype)[None]
    y, da, one = torch.empty_like(z), torch.empty_like(z), torch.ones_like(z)
    ch.Gated(y, z, act="gelu")
    ch.GatedBackward(da, None, one, z, act="gelu")
    v = z.to(O.F64)
    rel = 2.0 ** -15 if dtype != F32 else 2.0 ** -23 * (v * v + 9)
    u = O.HALF_STEP[dtype]
    want = O.act(v, "gelu")
    assert_within("gelu", y, want, (u + rel) * want.abs() + O.TINY[dtype])
    # The slope is Phi - |z| phi: at most 1.3 times its size in each.
    slope = O.dact(v, "gelu")
    assert_within("slope", da, slope, (u + 2 * rel) * slope.abs() + O.TINY[dtype])


def test_the_largest_number_restores_to_a_finite_one():
    top = torch.finfo(F32).max
    x = torch.zeros(3, 64, device="cuda")
    x[0, 3], x[1, 40], x[2] = top, -top, top
    x[0, 4] = top / 2
    for block in ch.BLOCKS:
        kept = ch.NewCheckpoint(x, block)
        back = torch.empty_like(x)
        ch.Pack8(kept, x)
        ch.Unpack8(back, kept)
        assert torch.isfinite(back).all()
        step = kept.scales.repeat_interleave(block, 1)[:, :64].to(O.F64)
        assert_within("restored", back, x.to(O.F64), step * 0.50002)
        assert kept.codes[0, 3] == 127 and kept.codes[1, 40] == -127 and (kept.codes[2] == 127).all()


def test_calls_without_elements_by_any_axis():
    for shape in ((2, 0, 8), (0, 3, 8), (2, 0, 4, 8), (2, 3, 0, 8)):
        x = torch.empty(*shape, device="cuda")
        y, dx, k = torch.empty_like(x), torch.empty_like(x), ch.NewCheckpoint(x, 32)
        mean, rstd = torch.ones(2, shape[0], 2, device="cuda")
        dw, db = torch.ones(2, 8, device="cuda")
        ch.GroupNorm(y, x, groups=2, mean=mean, rstd=rstd, ckpt=k)
        ch.GroupNormBackward(dx, dw, db, y, x, mean, rstd, groups=2)
        assert (mean == 0).all() and (dw == 0).all() and (db == 0).all()
        ch.Pack8(k, x)
        ch.Unpack8(y, k)
        ch.Gated(y, x, dx, a_ckpt=k)
        ch.GatedBackward(dx, None, y, x)


def test_memory_freed_after_a_call_on_another_stream_waits_for_it():
    """torch hands a freed tensor's memory to the next allocation unless it
    knows of the stream that still reads it."""
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream, C.c_void_p(side.cuda_stream)):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()   # no other memory of x's size is free
        x = torch.full((1, 4096, 4096), 0.5, device="cuda")
        y, kept = torch.empty_like(x), ch.NewCheckpoint(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)   # about a tenth of a second
        at = x.data_ptr()
        ch.GroupNorm(y, x, groups=32, ckpt=kept, stream=stream)
        del x
        other = torch.empty(1, 4096, 4096, device="cuda")
        assert other.data_ptr() != at
        torch.cuda.synchronize()


@pytest.mark.parametrize("before", ["nothing", "norm", "pack"])
def test_a_capture_after_calls_that_took_no_scratch(before):
    """A graph may hold calls that need scratch whether or not an earlier call
    of the process took any."""
    fresh_process(f"""
        import torch
        from simtgo_b200 import channels as ch
        g = torch.Generator(device="cuda").manual_seed(1)
        small = torch.randn(1, 8, 8, device="cuda", generator=g)
        if {before!r} == "norm":
            ch.GroupNorm(torch.empty_like(small), small, groups=1)
        elif {before!r} == "pack":
            ch.Pack8(ch.NewCheckpoint(small), small)
        x = torch.randn(1, 30000, 40, device="cuda", generator=g)
        y, dx = torch.zeros_like(x), torch.zeros_like(x)
        mean, rstd = torch.zeros(2, 1, 5, device="cuda")
        dw, db = torch.zeros(2, 40, device="cuda")

        def step():
            ch.GroupNorm(y, x, groups=5, mean=mean, rstd=rstd)
            ch.GroupNormBackward(dx, dw, db, x, x, mean, rstd, groups=5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, dx, dw, db)]
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, (y, dx, dw, db)))
        """)
