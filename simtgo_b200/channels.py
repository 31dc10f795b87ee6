"""Channels-last operators over libsimtgo_b200.so: group norm with an
activation, 8-bit activation checkpoints, and the gated unit, forward and
backward.

    kept = channels.NewCheckpoint(x)                       # codes and scales for x
    channels.GroupNorm(y, x, weight, bias, groups=32, act="silu",
                       mean=mean, rstd=rstd, ckpt=kept)    # x may be freed after this
    channels.GroupNormBackward(dx, dweight, dbias, dy, kept, mean, rstd, weight, bias,
                               groups=32, act="silu")
    channels.Pack8(kept, x); channels.Unpack8(x, kept)
    channels.Gated(y, a, b, act="silu", a_ckpt=ka, b_ckpt=kb)
    channels.GatedBackward(da, db, dy, ka, kb, act="silu")

Outputs come first, as in the kernels of package kernels, and are the caller's
CUDA tensors. Batches are [samples, positions, channels] or [samples, height,
width, channels] (a channels_last NCHW tensor after permute(0, 2, 3, 1)), rows
are any tensor whose last axis is the channels; the last axis has stride 1,
the others any strides that need no copy. Element types are float32, bfloat16
and float16. Calls are queued on `stream`, or on torch's current stream of the
tensors' device, and not waited for; a tensor may be freed after the call on
either. Nothing here records an autograd graph.

No counterpart in the reference; they stand beside Softclip, Quantize and
WarpReduceSum (kernels/softclip.go:11, quantize.go:16, warpreduce.go:21).
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import check

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"none": 0, "silu": 1, "gelu": 2, "softclip": 3}
BLOCKS = (32, 64, 128, 256)


class Checkpoint:
    """The 8-bit checkpoint of a tensor: int8 codes in the tensor's shape and a
    float32 scale for each `block` consecutive channels of a row, shaped
    [..., ceil(channels/block)]."""

    __slots__ = ("codes", "scales", "block")

    def __init__(self, codes, scales, block=128):
        self.codes, self.scales, self.block = codes, scales, block


def NewCheckpoint(x, block=128):
    """Room for the checkpoint of x (uninitialised)."""
    if block not in BLOCKS:
        raise ValueError(f"channels: a checkpoint block is one of {BLOCKS}, got {block}")
    shape = x.shape
    return Checkpoint(torch.empty(shape, dtype=torch.int8, device=x.device),
                      torch.empty(*shape[:-1], -(-shape[-1] // block), dtype=torch.float32,
                                  device=x.device), block)


def _type(t, name):
    k = _TYPES.get(t.dtype)
    if k is None:
        raise TypeError(f"channels: {name} is {t.dtype}; float32, bfloat16 and float16 are taken")
    return k


def _same(t, like, name, other):
    """t has like's shape, type and device."""
    if t.shape != like.shape:
        raise _lib.LengthError(_lib.ELENGTH, f"channels: {name} has shape {tuple(t.shape)}, "
                                             f"{other} {tuple(like.shape)}")
    if t.dtype is not like.dtype:
        raise TypeError(f"channels: {name} is {t.dtype}, {other} {like.dtype}")
    if t.get_device() != like.get_device():   # the CPU is device -1
        raise ValueError(f"channels: {name} is on {t.device}, the call on {like.device}")


def _flat(t, like, numel, dtype, name):
    """The address of a contiguous array of numel elements (None: no array)."""
    if t is None:
        return None
    if (t.dtype is dtype and t.numel() == numel and t.is_contiguous()
            and t.get_device() == like.get_device()):
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"channels: {name} is {t.dtype}, the kernel takes {dtype}")
    if t.numel() != numel:
        raise _lib.LengthError(_lib.ELENGTH, f"channels: {name} has {t.numel()} elements, the "
                                             f"call takes {numel}")
    if not t.is_contiguous():
        raise TypeError(f"channels: {name} must be contiguous")
    raise ValueError(f"channels: {name} is on {t.device}, the call on {like.device}")


def _kept(k, like, name):
    """Addresses of a checkpoint's arrays for a tensor shaped like `like`."""
    if k.block not in BLOCKS:
        raise ValueError(f"channels: a checkpoint block is one of {BLOCKS}, got {k.block}")
    c = like.shape[-1]
    n = like.numel()
    blocks = n // c * -(-c // k.block) if c else 0
    return (_flat(k.codes, like, n, torch.int8, name + ".codes"),
            _flat(k.scales, like, blocks, torch.float32, name + ".scales"))


def _batch(t, name):
    """(sample pitch, row pitch) of a batch of rows."""
    sh, st = t.shape, t.stride()
    if len(sh) != 3 and len(sh) != 4:
        raise TypeError(f"channels: {name} is a batch [samples, positions, channels] or "
                        f"[samples, height, width, channels], got {tuple(sh)}")
    if st[-1] != 1 and sh[-1] > 1:
        raise TypeError(f"channels: the channels of {name} must be adjacent (stride 1)")
    if len(sh) == 3:
        return st[0], st[1]
    if sh[2] == 1:
        return st[0], st[1]
    if t.numel() and sh[1] > 1 and st[1] != sh[2] * st[2]:
        raise TypeError(f"channels: the height and width of {name} must lie as one axis of rows")
    return st[0], st[2]


def _rows(t, name):
    """The pitch of a tensor's rows, all its axes but the last taken as one."""
    st = t.stride()
    if len(st) == 2 and st[1] == 1:
        return st[0]
    sh = t.shape
    if not sh:
        raise TypeError(f"channels: {name} has no channels")
    if st[-1] != 1 and sh[-1] > 1:
        raise TypeError(f"channels: the channels of {name} must be adjacent (stride 1)")
    if len(sh) == 1:
        return sh[0]
    if len(sh) == 2 or not t.numel():
        return st[-2]
    pitch = run = None
    for n, s in zip(reversed(sh[:-1]), reversed(st[:-1])):
        if n == 1:
            continue
        if pitch is None:
            pitch, run = s, s * n
        elif s == run:
            run *= n
        else:
            raise TypeError(f"channels: the rows of {name} must lie one pitch apart")
    return sh[-1] if pitch is None else pitch


def _extent(v, what):
    """v, an extent that the library takes in 32 bits: ctypes would wrap it."""
    if v > 0x7fffffff:
        raise _lib.SimtgoError(_lib.ESIZE, f"channels: {v} {what}, at most {0x7fffffff}")
    return v


def _matrix(t):
    """(rows, channels) of a tensor of rows."""
    c = _extent(t.shape[-1], "channels")
    return t.numel() // c if c else 0, c


def _act(act):
    k = ACTS.get(act)
    if k is None:
        raise ValueError(f"channels: no activation {act!r}; there are {', '.join(ACTS)}")
    return k


# Configurations by their values alone (numbers: a tensor would be known by its
# identity); the library copies one before it returns.
@functools.lru_cache(maxsize=256)
def _norm_cfg(*v):
    c = _lib.GroupNormConfig(*v)
    return c, C.byref(c)


@functools.lru_cache(maxsize=256)
def _gated_cfg(*v):
    c = _lib.GatedUnitConfig(*v)
    return c, C.byref(c)


# torch.cuda.current_device() and current_stream(dev).cuda_stream, without the
# objects they build: a call on a few rows lasts a few microseconds.
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(name, dev, stream, tensors, *args):
    """Runs the library's function on device dev, on the caller's stream or on
    torch's current one. On another stream than the current one the tensors'
    memory is kept from new tensors until the call is done there."""
    if stream is None:
        sp = _raw_stream(dev)
    else:
        sp = getattr(stream, "cuda_stream", stream)
        sp = getattr(sp, "value", sp) or 0   # a ctypes pointer
    fn = getattr(_lib._lib or _lib.load(), name)
    if dev == _device():
        rc = fn(*args, sp)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, sp)
    if rc:
        check(rc)
    if stream is not None and sp != _raw_stream(dev):
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(sp, device=dev)
        for t in tensors:
            for v in (t.codes, t.scales) if isinstance(t, Checkpoint) else (t,):
                if v is not None:
                    v.record_stream(stream)


def _on_gpu(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"channels: {name} must be a CUDA tensor")
    return t.get_device()


def _norm_args(like, groups, weight, bias, mean, rstd, lengths):
    sh = like.shape
    n, c = _extent(sh[0], "samples"), _extent(sh[-1], "channels")
    s = _extent(sh[1] if len(sh) == 3 else sh[1] * sh[2], "positions")
    if not isinstance(groups, int) or groups <= 0 or c % groups:
        raise ValueError(f"channels: {c} channels are not a whole number of {groups} groups")
    p = weight if weight is not None else bias
    pt = 0 if p is None else _type(p, "weight" if weight is not None else "bias")
    pd = None if p is None else p.dtype
    return (n, s, c, pt, _flat(weight, like, c, pd, "weight"), _flat(bias, like, c, pd, "bias"),
            _flat(mean, like, n * groups, torch.float32, "mean"),
            _flat(rstd, like, n * groups, torch.float32, "rstd"),
            _flat(lengths, like, n, torch.int32, "lengths"))


def GroupNorm(y, x, weight=None, bias=None, *, groups, eps=1e-5, act="none", threshold=1.0,
              mean=None, rstd=None, lengths=None, ckpt=None, stream=None):
    """y = act((x - mean)*rstd*weight + bias), mean and rstd = 1/sqrt(var + eps)
    over each group of channels of a sample's valid positions.

    weight and bias hold one value per channel (one type; None: ones, zeros).
    mean and rstd, float32 [samples, groups], receive the statistics the
    backward pass reads. lengths, int32 [samples], gives each sample's valid
    positions: later ones are neither read nor written. ckpt receives the 8-bit
    checkpoint of x in the same pass. threshold belongs to act="softclip"."""
    dev = _on_gpu(x, "x")
    _same(y, x, "y", "x")
    xs, xr = _batch(x, "x")
    ys, yr = _batch(y, "y")
    n, s, c, pt, w, b, mu, rs, ln = _norm_args(x, groups, weight, bias, mean, rstd, lengths)
    codes = scales = None
    block = 0
    if ckpt is not None:
        codes, scales = _kept(ckpt, x, "ckpt")
        block = ckpt.block
    cfg = _norm_cfg(xs, xr, ys, yr, 0, 0, n, s, c, groups, _type(x, "x"), pt, _act(act), block,
                    float(threshold), float(eps))[1]
    _call("simtgo_GroupNorm", dev, stream, (y, x, weight, bias, mean, rstd, lengths, ckpt),
          y.data_ptr(), mu, rs, x.data_ptr(), w, b, ln, codes, scales, cfg)


def GroupNormBackward(dx, dweight, dbias, dy, x, mean, rstd, weight=None, bias=None, *, groups,
                      eps=1e-5, act="none", threshold=1.0, lengths=None, stream=None):
    """The gradients of GroupNorm from its mean and rstd; x is its input or the
    Checkpoint it filled. dweight and dbias (float32, per channel) are
    overwritten with sums over all samples and valid positions; dx, dweight and
    dbias may each be None."""
    dev = _on_gpu(dy, "dy")
    ys, yr = _batch(dy, "dy")
    if mean is None or rstd is None:
        raise TypeError("channels: the backward pass needs mean and rstd")
    n, s, c, pt, w, b, mu, rs, ln = _norm_args(dy, groups, weight, bias, mean, rstd, lengths)
    xp = codes = scales = dp = None
    xs = xr = ds = dr = block = 0
    if isinstance(x, Checkpoint):
        codes, scales = _kept(x, dy, "x")
        block = x.block
    else:
        _same(x, dy, "x", "dy")
        xs, xr = _batch(x, "x")
        xp = x.data_ptr()
    if dx is not None:
        _same(dx, dy, "dx", "dy")
        ds, dr = _batch(dx, "dx")
        dp = dx.data_ptr()
    cfg = _norm_cfg(xs, xr, ys, yr, ds, dr, n, s, c, groups, _type(dy, "dy"), pt, _act(act), block,
                    float(threshold), float(eps))[1]
    _call("simtgo_GroupNorm_backward", dev, stream,
          (dx, dweight, dbias, dy, x, mean, rstd, weight, bias, lengths), dp,
          _flat(dweight, dy, c, torch.float32, "dweight"),
          _flat(dbias, dy, c, torch.float32, "dbias"), dy.data_ptr(), xp, codes, scales, mu, rs,
          w, b, ln, cfg)


def Pack8(ckpt, x, *, stream=None):
    """Writes the 8-bit checkpoint of x: per block of channels a scale, the
    largest magnitude over 127, and codes rounded to the nearest multiple of
    it. A block with a NaN or an infinity restores to NaN."""
    dev = _on_gpu(x, "x")
    pitch = _rows(x, "x")
    codes, scales = _kept(ckpt, x, "ckpt")
    rows, c = _matrix(x)
    _call("simtgo_Pack8", dev, stream, (ckpt, x), codes, scales, x.data_ptr(), _type(x, "x"), rows,
          c, pitch, ckpt.block)


def Unpack8(x, ckpt, *, stream=None):
    """x = code * scale, rounded to x's type."""
    dev = _on_gpu(x, "x")
    pitch = _rows(x, "x")
    codes, scales = _kept(ckpt, x, "ckpt")
    rows, c = _matrix(x)
    _call("simtgo_Unpack8", dev, stream, (x, ckpt), x.data_ptr(), codes, scales, _type(x, "x"),
          rows, c, pitch, ckpt.block)


def Gated(y, a, b=None, *, act="silu", threshold=1.0, a_ckpt=None, b_ckpt=None, stream=None):
    """y = act(a)*b, or act(a) without b; a_ckpt and b_ckpt receive the 8-bit
    checkpoints of a and b in the same pass."""
    dev = _on_gpu(a, "a")
    _same(y, a, "y", "a")
    ap, bp, yp = _rows(a, "a"), 0, _rows(y, "y")
    bd = ac = asc = bc = bsc = None
    block = 0
    if b is not None:
        _same(b, a, "b", "a")
        bp = _rows(b, "b")
        bd = b.data_ptr()
    if a_ckpt is not None:
        ac, asc = _kept(a_ckpt, a, "a_ckpt")
        block = a_ckpt.block
    if b_ckpt is not None:
        if b is None:
            raise ValueError("channels: a checkpoint of b, but no b")
        if block and b_ckpt.block != block:
            raise ValueError("channels: both checkpoints have the same block")
        bc, bsc = _kept(b_ckpt, a, "b_ckpt")
        block = b_ckpt.block
    rows, c = _matrix(a)
    cfg = _gated_cfg(rows, ap, bp, yp, 0, 0, c, _type(a, "a"), _act(act), block,
                     float(threshold), 0)[1]
    _call("simtgo_Gated", dev, stream, (y, a, b, a_ckpt, b_ckpt), y.data_ptr(), a.data_ptr(), bd,
          ac, asc, bc, bsc, cfg)


def GatedBackward(da, db, dy, a, b=None, *, act="silu", threshold=1.0, stream=None):
    """da = dy*b*act'(a) and db = dy*act(a); a and b are tensors, or both
    Checkpoints. da and db may each be None."""
    dev = _on_gpu(dy, "dy")
    yp = _rows(dy, "dy")
    src = []
    block = 0
    if b is not None and isinstance(a, Checkpoint) != isinstance(b, Checkpoint):
        raise TypeError("channels: a and b are both tensors or both checkpoints")
    for t, name in ((a, "a"), (b, "b")):
        if t is None:
            src.append((None, None, None, 0))
        elif isinstance(t, Checkpoint):
            if block and t.block != block:
                raise ValueError("channels: both checkpoints have the same block")
            block = t.block
            src.append((None, *_kept(t, dy, name), 0))
        else:
            _same(t, dy, name, "dy")
            src.append((t.data_ptr(), None, None, _rows(t, name)))
    out = []
    for t, name in ((da, "da"), (db, "db")):
        if t is None:
            out.append((None, 0))
        else:
            _same(t, dy, name, "dy")
            out.append((t.data_ptr(), _rows(t, name)))
    (ad, ac, asc, ap), (bd, bc, bsc, bp) = src
    rows, c = _matrix(dy)
    cfg = _gated_cfg(rows, ap, bp, yp, out[0][1], out[1][1], c, _type(dy, "dy"), _act(act), block,
                     float(threshold), 0)[1]
    _call("simtgo_Gated_backward", dev, stream, (da, db, dy, a, b), out[0][0], out[1][0],
          dy.data_ptr(), ad, bd, ac, asc, bc, bsc, cfg)


__all__ = ["Checkpoint", "NewCheckpoint", "GroupNorm", "GroupNormBackward", "Pack8", "Unpack8",
           "Gated", "GatedBackward", "ACTS", "BLOCKS"]
