"""Thin tensor-level wrappers over the single-operator C entry points.

Activations are torch tensors in the library's layout: NHWC ``(B, H, W, Cpad)`` with
``Cpad = pad_ch(C)`` and dtype ``torch.float32`` or ``torch.bfloat16``.  Parameters and
parameter gradients are fp32 in the reference's layouts.  Every function enqueues on the
current torch stream and returns torch tensors it allocated; nothing here computes
with torch ops."""
from __future__ import annotations

import ctypes
import functools
import operator
from typing import Optional, Tuple

import torch

from ._lib import MI_ACT_GELU, MI_ACT_NONE, MI_ACT_RELU, MI_ACT_SILU, MI_BF16, MI_F32, check, lib
from ._lib import Dropout as _DropoutDesc


def pad_ch(c: int) -> int:
    """Stored channel count of a C-channel tensor (same rule as ``mi_pad_channels``)."""
    return 32 if c <= 32 else (c + 15) // 16 * 16


def mi_dtype(dt: torch.dtype) -> int:
    if dt == torch.float32:
        return MI_F32
    if dt == torch.bfloat16:
        return MI_BF16
    raise TypeError(f"unsupported compute dtype {dt}: use torch.float32 or torch.bfloat16")


def torch_dtype(name) -> torch.dtype:
    if isinstance(name, torch.dtype):
        return name
    table = {"fp32": torch.float32, "float32": torch.float32, "f32": torch.float32,
             "bf16": torch.bfloat16, "bfloat16": torch.bfloat16}
    try:
        return table[str(name).lower()]
    except KeyError:
        raise ValueError(f"unknown compute dtype {name!r} (fp32 or bf16)") from None


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("this operator runs only as a HIP kernel on the GPU; got a CPU tensor "
                               "(there is no CPU fallback)")


def _view(t: torch.Tensor, coff: int = 0) -> Tuple[int, int, int]:
    """(pointer, channel stride, channel offset) of an NHWC tensor."""
    assert t.dim() == 4 and t.is_contiguous()
    return t.data_ptr(), t.shape[3], coff


# ------------------------------------------------------------------ layout
def to_nhwc(x: torch.Tensor, dtype=torch.float32, out: Optional[torch.Tensor] = None, coff: int = 0):
    _need_cuda(x)
    x = x.contiguous().float()
    B, Cc, H, W = x.shape
    if out is None:
        out = torch.empty((B, H, W, pad_ch(Cc)), device=x.device, dtype=dtype)
    check(lib().mi_nchw_to_nhwc(x.data_ptr(), out.data_ptr(), out.shape[3], coff, B, Cc, H, W,
                                mi_dtype(out.dtype), _stream()), "nchw_to_nhwc")
    return out


def from_nhwc(t: torch.Tensor, channels: int, coff: int = 0) -> torch.Tensor:
    _need_cuda(t)
    B, H, W, cs = t.shape
    out = torch.empty((B, channels, H, W), device=t.device, dtype=torch.float32)
    check(lib().mi_nhwc_to_nchw(t.data_ptr(), cs, coff, out.data_ptr(), B, channels, H, W,
                                mi_dtype(t.dtype), _stream()), "nhwc_to_nchw")
    return out


# ------------------------------------------------------------------ packing
def pack_conv3x3(weight: torch.Tensor, dtype, split: int = 0, want_bwd: bool = True):
    _need_cuda(weight)
    Cout, Cin = weight.shape[:2]
    L, dt = lib(), mi_dtype(dtype)
    es = 2 if dtype == torch.bfloat16 else 4
    wf = torch.empty(L.mi_packed_conv3x3_bytes(Cout, Cin, split, dt, 0) // es, device=weight.device, dtype=dtype)
    wb = torch.empty(L.mi_packed_conv3x3_bytes(Cout, Cin, split, dt, 1) // es, device=weight.device,
                     dtype=dtype) if want_bwd else None
    check(L.mi_pack_conv3x3(weight.contiguous().data_ptr(), wf.data_ptr(), wb.data_ptr() if want_bwd else None,
                            Cout, Cin, split, dt, _stream()), "pack_conv3x3")
    return wf, wb


def pack_convt2x2(weight: torch.Tensor, dtype, want_bwd: bool = True):
    _need_cuda(weight)
    Cin, Cout = weight.shape[:2]
    L, dt = lib(), mi_dtype(dtype)
    es = 2 if dtype == torch.bfloat16 else 4
    wf = torch.empty(L.mi_packed_convt2x2_bytes(Cin, Cout, dt, 0) // es, device=weight.device, dtype=dtype)
    wb = torch.empty(L.mi_packed_convt2x2_bytes(Cin, Cout, dt, 1) // es, device=weight.device,
                     dtype=dtype) if want_bwd else None
    check(L.mi_pack_convt2x2(weight.contiguous().data_ptr(), wf.data_ptr(), wb.data_ptr() if want_bwd else None,
                             Cin, Cout, dt, _stream()), "pack_convt2x2")
    return wf, wb


# ------------------------------------------------------------------ 3x3 conv
def conv3x3_relu_fwd(x, wfwd, bias, Cin, Cout, split=0, relu=True, out=None, out_coff=0):
    B, H, W, _ = x.shape
    if out is None:
        out = torch.empty((B, H, W, pad_ch(Cout)), device=x.device, dtype=x.dtype)
    check(lib().mi_conv3x3_relu_fwd(*_view(x), wfwd.data_ptr(), bias.data_ptr(), *_view(out, out_coff),
                                    B, H, W, Cin, split, Cout, int(relu), mi_dtype(x.dtype), _stream()), "conv3x3_fwd")
    return out


def conv3x3_dgrad(dy, wbwd, Cin, Cout, split=0, mask=None, dy_coff=0):
    B, H, W, _ = dy.shape
    cp = pad_ch(split) + pad_ch(Cin - split) if split else pad_ch(Cin)
    dx = torch.empty((B, H, W, cp), device=dy.device, dtype=dy.dtype)
    mv = _view(mask) if mask is not None else (None, 0, 0)
    check(lib().mi_conv3x3_dgrad(*_view(dy, dy_coff), wbwd.data_ptr(), *_view(dx), *mv,
                                 B, H, W, Cin, split, Cout, mi_dtype(dy.dtype), _stream()), "conv3x3_dgrad")
    return dx


def conv3x3_wgrad(x, dy, Cin, Cout, split=0, dW=None, db=None, alpha=1.0, beta=0.0, dy_coff=0):
    B, H, W, _ = x.shape
    dt = mi_dtype(x.dtype)
    if dW is None:
        dW = torch.empty((Cout, Cin, 3, 3), device=x.device, dtype=torch.float32)
        db = torch.empty((Cout,), device=x.device, dtype=torch.float32)
    nbytes = lib().mi_conv3x3_wgrad_ws_bytes(B, H, W, Cin, split, Cout, dt)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    check(lib().mi_conv3x3_wgrad(*_view(x), *_view(dy, dy_coff), dW.data_ptr(), db.data_ptr(), alpha, beta,
                                 ws.data_ptr(), nbytes, B, H, W, Cin, split, Cout, dt, _stream()), "conv3x3_wgrad")
    return dW, db


# ------------------------------------------------------------------ max-pool
def maxpool2_fwd(x, C, x_coff=0):
    B, H, W, _ = x.shape
    y = torch.empty((B, H // 2, W // 2, pad_ch(C)), device=x.device, dtype=x.dtype)
    check(lib().mi_maxpool2_fwd(*_view(x, x_coff), *_view(y), B, H, W, C, mi_dtype(x.dtype), _stream()), "maxpool2_fwd")
    return y


def maxpool2_bwd(x, dy_pool, C, dskip=None, relu_mask=False, x_coff=0):
    B, H, W, _ = x.shape
    dx = torch.empty((B, H, W, pad_ch(C)), device=x.device, dtype=x.dtype)
    sv = _view(dskip) if dskip is not None else (None, 0, 0)
    check(lib().mi_maxpool2_bwd(*_view(x, x_coff), *_view(dy_pool), *sv, *_view(dx), B, H, W, C, int(relu_mask),
                                mi_dtype(x.dtype), _stream()), "maxpool2_bwd")
    return dx


# ------------------------------------------------------------------ transposed conv
def convt2x2_fwd(x, wfwd, bias, Cin, Cout, out=None, out_coff=0):
    B, H, W, _ = x.shape
    if out is None:
        out = torch.empty((B, 2 * H, 2 * W, pad_ch(Cout)), device=x.device, dtype=x.dtype)
    check(lib().mi_convt2x2_fwd(*_view(x), wfwd.data_ptr(), bias.data_ptr(), *_view(out, out_coff), B, H, W, Cin, Cout,
                                mi_dtype(x.dtype), _stream()), "convt2x2_fwd")
    return out


def convt2x2_dgrad(dy, wbwd, Cin, Cout, mask=None, dy_coff=0):
    B, H2, W2, _ = dy.shape
    H, W = H2 // 2, W2 // 2
    dx = torch.empty((B, H, W, pad_ch(Cin)), device=dy.device, dtype=dy.dtype)
    mv = _view(mask) if mask is not None else (None, 0, 0)
    check(lib().mi_convt2x2_dgrad(*_view(dy, dy_coff), wbwd.data_ptr(), *_view(dx), *mv, B, H, W, Cin, Cout,
                                  mi_dtype(dy.dtype), _stream()), "convt2x2_dgrad")
    return dx


def convt2x2_wgrad(x, dy, Cin, Cout, alpha=1.0, beta=0.0, dy_coff=0):
    B, H, W, _ = x.shape
    dt = mi_dtype(x.dtype)
    dW = torch.empty((Cin, Cout, 2, 2), device=x.device, dtype=torch.float32)
    db = torch.empty((Cout,), device=x.device, dtype=torch.float32)
    nbytes = lib().mi_convt2x2_wgrad_ws_bytes(B, H, W, Cin, Cout, dt)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    check(lib().mi_convt2x2_wgrad(*_view(x), *_view(dy, dy_coff), dW.data_ptr(), db.data_ptr(), alpha, beta,
                                  ws.data_ptr(), nbytes, B, H, W, Cin, Cout, dt, _stream()), "convt2x2_wgrad")
    return dW, db


# ------------------------------------------------------------------ head
def head_fwd(x, weight, bias, Cin, Cout):
    B, H, W, _ = x.shape
    pred = torch.empty((B, Cout, H, W), device=x.device, dtype=torch.float32)
    check(lib().mi_conv1x1_head_fwd(*_view(x), weight.data_ptr(), bias.data_ptr(), pred.data_ptr(), B, H, W, Cin, Cout,
                                    mi_dtype(x.dtype), _stream()), "head_fwd")
    return pred


def head_bwd(x, weight, dpred, Cin, Cout, relu_mask=True, alpha=1.0, beta=0.0):
    B, H, W, _ = x.shape
    dx = torch.empty_like(x)
    dW = torch.empty((Cout, Cin, 1, 1), device=x.device, dtype=torch.float32)
    db = torch.empty((Cout,), device=x.device, dtype=torch.float32)
    nbytes = lib().mi_conv1x1_head_ws_bytes(Cin, Cout)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    check(lib().mi_conv1x1_head_bwd(*_view(x), weight.data_ptr(), dpred.contiguous().data_ptr(), *_view(dx),
                                    dW.data_ptr(), db.data_ptr(), alpha, beta, ws.data_ptr(), nbytes, B, H, W, Cin, Cout,
                                    int(relu_mask), mi_dtype(x.dtype), _stream()), "head_bwd")
    return dx, dW, db


# ------------------------------------------------------------------ dropout, group norm
ACTIVATIONS = {"none": MI_ACT_NONE, "relu": MI_ACT_RELU, "silu": MI_ACT_SILU, "gelu": MI_ACT_GELU}


class Drop:
    """What is dropped: a function of these values and of an element's place alone, so no mask is stored and the
    backward pass takes the same object.

    ``p`` counts in steps of 2^-16 (survivors are scaled by the rounded value).  ``seed`` and ``offset`` are integers
    in [0, 2^64); layers of one step take different offsets (or seeds).  ``offset_dev`` (a one-element int64 tensor on
    the GPU) is added to ``offset`` when a kernel runs: a captured graph replays with new masks if it is counted up
    between replays.  ``per_channel`` drops whole feature maps.  A ``Drop`` is fixed once it is made: a backward pass that is
    still to come needs it as it was."""

    __slots__ = ("_p", "_seed", "_offset", "_offset_dev", "_per_channel", "_desc")
    p, seed, offset, offset_dev, per_channel = (property(operator.attrgetter(n)) for n in __slots__[:-1])

    def __init__(self, p: float, seed: int, offset: int = 0, offset_dev: Optional[torch.Tensor] = None,
                 per_channel: bool = False):
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout: p must be between 0 and 1, got {p}")
        if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
            raise ValueError("dropout: seed and offset must be in [0, 2^64)")
        if offset_dev is not None and (offset_dev.dtype != torch.int64 or offset_dev.numel() != 1 or not offset_dev.is_cuda):
            raise ValueError("dropout: offset_dev must be a one-element int64 tensor on the GPU")
        self._p, self._seed, self._offset, self._offset_dev, self._per_channel = p, seed, offset, offset_dev, per_channel
        self._desc = _DropoutDesc(p, seed, offset, offset_dev.data_ptr() if offset_dev is not None else None, int(per_channel))


def _drop_ref(drop: Optional[Drop], dev: torch.device):
    if drop is None:
        return None
    if drop._offset_dev is not None and drop._offset_dev.device != dev:
        raise RuntimeError(f"dropout: offset_dev is on {drop._offset_dev.device}, the activation on {dev}")
    return ctypes.byref(drop._desc)


def _nhwc(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None) -> None:
    """Refuses what is no dense (B, H, W, channels) activation, or not of the size, type and device of ``like``."""
    if not t.is_cuda:
        _need_cuda(t)
    if t.dim() != 4 or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous (B, H, W, channels) tensor, got shape {tuple(t.shape)}, strides {t.stride()}")
    if like is not None and (t.shape[:3] != like.shape[:3] or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{what}: {tuple(t.shape[:3])} {t.dtype} on {t.device} does not go with "
                         f"{tuple(like.shape[:3])} {like.dtype} on {like.device}")


def _channel_vector(t: Optional[torch.Tensor], n: int, dev: torch.device, what: str):
    """Pointer of an fp32 tensor of n values on ``dev`` (None stays None)."""
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != n or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{what}: expected {n} contiguous float32 values on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


class _NoGuard:
    __slots__ = ()

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def _on(dev: torch.device):
    """Context in which kernels are launched on ``dev``; free when it is the current device already."""
    return _NO_GUARD if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _activation(act: str) -> int:
    try:
        return ACTIVATIONS[act]
    except KeyError:
        raise ValueError(f"unknown activation {act!r} ({', '.join(ACTIVATIONS)})") from None


@functools.lru_cache(maxsize=256)
def _norm_ws_bytes(B, H, W, Cc, groups, backward, dt) -> int:
    return lib().mi_group_norm_ws_bytes(B, H, W, Cc, groups, backward, dt)


def _new_activation(x: torch.Tensor, C: int) -> torch.Tensor:
    """An activation of C channels with the size, type and device of ``x``."""
    B, H, W, cs = x.shape
    width = pad_ch(C)
    return torch.empty_like(x) if width == cs else x.new_empty((B, H, W, width))


# The small calls of these layers are bound by the host: ``torch.cuda.current_stream`` builds an object (1.8 us), this
# returns the handle alone (0.1 us).
_raw_stream = torch._C._cuda_getCurrentRawStream
_POLLS = -1                  # see mi_group_norm_act_fwd


def dropout_fwd(x, C, drop: Optional[Drop], residual=None, x_coff=0, residual_coff=0, out=None, out_coff=0):
    """``residual + dropout(x)`` (NHWC, C of the channels from ``x_coff`` on); ``out`` may be x or the residual;
    without a ``drop`` nothing is dropped."""
    _nhwc(x, "dropout")
    B, H, W, cs = x.shape
    dev, dt = x.device, mi_dtype(x.dtype)
    if residual is None:
        rp, rcs = None, 0
    else:
        _nhwc(residual, "dropout residual", x)
        rp, rcs = residual.data_ptr(), residual.shape[3]
    with _on(dev):
        if out is None:
            out = _new_activation(x, C)
        else:
            _nhwc(out, "dropout out", x)
        check(lib().mi_dropout_fwd(x.data_ptr(), cs, x_coff, rp, rcs, residual_coff, out.data_ptr(), out.shape[3], out_coff, B, H, W,
                                   C, _drop_ref(drop, dev), dt, _raw_stream(dev.index)), "dropout_fwd")
    return out


def dropout_bwd(dy, C, drop: Drop, dy_coff=0, out=None, out_coff=0):
    """Gradient with respect to x (that of the residual is dy itself)."""
    return dropout_fwd(dy, C, drop, x_coff=dy_coff, out=out, out_coff=out_coff)


def group_norm_act_fwd(x, C, groups, weight=None, bias=None, act="none", eps=1e-5, drop: Optional[Drop] = None, x_coff=0,
                       out=None, out_coff=0):
    """``dropout(act(group_norm(x)))`` of the C channels from ``x_coff`` on.  Returns (y, mean, rstd): the statistics
    (B, groups) are what the backward pass needs besides x."""
    _nhwc(x, "group_norm_act")
    B, H, W, cs = x.shape
    dev, dt = x.device, mi_dtype(x.dtype)
    code = _activation(act)
    wp, bp = _channel_vector(weight, C, dev, "group_norm_act weight"), _channel_vector(bias, C, dev, "group_norm_act bias")
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm_act: {C} channels do not split into {groups} groups")
    with _on(dev):
        if out is None:
            out = _new_activation(x, C)
        else:
            _nhwc(out, "group_norm_act out", x)
        mean, rstd = torch.empty((2, B, groups), device=dev, dtype=torch.float32).unbind()
        nbytes = _norm_ws_bytes(B, H, W, C, groups, 0, dt)
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
        check(lib().mi_group_norm_act_fwd(x.data_ptr(), cs, x_coff, wp, bp, out.data_ptr(), out.shape[3], out_coff, mean.data_ptr(),
                                          rstd.data_ptr(), B, H, W, C, groups, code, eps, _drop_ref(drop, dev), _POLLS,
                                          ws.data_ptr() if nbytes else None, nbytes, dt, _raw_stream(dev.index)), "group_norm_act_fwd")
    return out, mean, rstd


def group_norm_act_bwd(x, dy, mean, rstd, C, groups, weight=None, bias=None, act="none", drop: Optional[Drop] = None, x_coff=0,
                       dy_coff=0, dweight=None, dbias=None, alpha=1.0, beta=0.0, want_dweight=True, want_dbias=True):
    """(dx, dweight, dbias) from what the forward pass was given and returned.  ``dweight`` / ``dbias`` are None where
    the parameter is, or is not wanted; tensors passed in receive ``alpha * gradient + beta * themselves``."""
    _nhwc(x, "group_norm_act")
    _nhwc(dy, "group_norm_act dy", x)
    B, H, W, cs = x.shape
    dev, dt = x.device, mi_dtype(x.dtype)
    code = _activation(act)
    wp, bp = _channel_vector(weight, C, dev, "group_norm_act weight"), _channel_vector(bias, C, dev, "group_norm_act bias")
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm_act: {C} channels do not split into {groups} groups")
    mp, rp = (_channel_vector(t, B * groups, dev, "group_norm_act statistics") for t in (mean, rstd))
    with _on(dev):
        dx = _new_activation(x, C)
        if weight is not None and dweight is None and want_dweight:
            dweight = torch.empty_like(weight) if beta == 0.0 else torch.zeros_like(weight)
        if bias is not None and dbias is None and want_dbias:
            dbias = torch.empty_like(bias) if beta == 0.0 else torch.zeros_like(bias)
        gp, hp = _channel_vector(dweight, C, dev, "group_norm_act dweight"), _channel_vector(dbias, C, dev, "group_norm_act dbias")
        nbytes = _norm_ws_bytes(B, H, W, C, groups, 1, dt)
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
        check(lib().mi_group_norm_act_bwd(x.data_ptr(), cs, x_coff, dy.data_ptr(), dy.shape[3], dy_coff, wp, bp, mp, rp,
                                          dx.data_ptr(), dx.shape[3], 0, gp, hp, alpha, beta, B, H, W, C, groups, code,
                                          _drop_ref(drop, dev), _POLLS, ws.data_ptr() if nbytes else None, nbytes, dt,
                                          _raw_stream(dev.index)), "group_norm_act_bwd")
    return dx, dweight, dbias


# ------------------------------------------------------------------ loss
def mse_fwd_bwd(pred, target, want_grad=True, gscale=1.0, gscale_dev: Optional[torch.Tensor] = None, want_sums=True):
    """Returns (out3, dpred): out3 = [mean sq err, sum |d|, sum d^2] (device fp32), or None without want_sums."""
    _need_cuda(pred, target)
    if pred.shape != target.shape:
        raise ValueError(f"mse: shape mismatch {tuple(pred.shape)} vs {tuple(target.shape)}")
    pred, target = pred.contiguous(), target.contiguous()
    n = pred.numel()
    out3 = torch.empty(3, device=pred.device, dtype=torch.float32) if want_sums else None
    dpred = torch.empty_like(pred) if want_grad else None
    nbytes = lib().mi_mse_ws_bytes(n)
    ws = torch.empty(nbytes, device=pred.device, dtype=torch.uint8)
    check(lib().mi_mse_fwd_bwd(pred.data_ptr(), target.data_ptr(), n, out3.data_ptr() if want_sums else None,
                               dpred.data_ptr() if want_grad else None, gscale,
                               gscale_dev.data_ptr() if gscale_dev is not None else None,
                               ws.data_ptr(), nbytes, _stream()), "mse")
    return out3, dpred


# ------------------------------------------------------------------ bilinear
def _strides_nchw(t):
    return t.stride(0), t.stride(1), t.stride(2), t.stride(3)


def bilinear_fwd_nchw(x: torch.Tensor, size) -> torch.Tensor:
    _need_cuda(x)
    x = x.contiguous()
    B, Cc, H, W = x.shape
    out = torch.empty((B, Cc, size[0], size[1]), device=x.device, dtype=x.dtype)
    check(lib().mi_bilinear_fwd(x.data_ptr(), *_strides_nchw(x), mi_dtype(x.dtype), out.data_ptr(), *_strides_nchw(out),
                                mi_dtype(out.dtype), B, Cc, H, W, size[0], size[1], _stream()), "bilinear_fwd")
    return out


def bilinear_bwd_nchw(dout: torch.Tensor, in_size) -> torch.Tensor:
    _need_cuda(dout)
    dout = dout.contiguous()
    B, Cc, Ho, Wo = dout.shape
    din = torch.empty((B, Cc, in_size[0], in_size[1]), device=dout.device, dtype=dout.dtype)
    check(lib().mi_bilinear_bwd(dout.data_ptr(), *_strides_nchw(dout), mi_dtype(dout.dtype), din.data_ptr(),
                                *_strides_nchw(din), mi_dtype(din.dtype), B, Cc, in_size[0], in_size[1], Ho, Wo,
                                _stream()), "bilinear_bwd")
    return din


# ------------------------------------------------------------------ optimiser
def adam_step(p, g, m, v, lr, beta1, beta2, eps, step, grad_scale=1.0):
    _need_cuda(p, g, m, v)
    check(lib().mi_adam_step(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(), lr, beta1, beta2, eps,
                             step, grad_scale, _stream()), "adam_step")
