"""Stand-alone operators on device tensors: the gated delta rule (a recurrence over frames with a matrix state) over whole clips and hop by
hop, and dense layers with 4-bit weights for a few rows -- the parts of a recurrent layer beside the engine's own (`dpdf_gated_delta`,
`dpdf_gated_delta_step`, `dpdf_w4_matvec`, `dpdf_w4_quantize` of include/dpdfnet_hip.h).

Tensors are torch tensors on one HIP device, float32, float16 or bfloat16; calls are queued on torch's current stream of that device,
allocate nothing beside their results (and, for a few long clips, a workspace) through torch and wait for nothing, so they can be captured into a graph.  Sums, states and accumulators are fp32
whatever the tensors' type.  There is no derivative: tensors that require a gradient are refused while gradients are recorded, and tensors that
carry a forward-mode tangent always.  Wrong types, shapes and overlaps raise ValueError, failures of the device RuntimeError."""
from __future__ import annotations

import ctypes
import math
import struct
from typing import TYPE_CHECKING, Optional, Tuple

from . import backend as _backend

if TYPE_CHECKING:  # pragma: no cover
    import torch

__all__ = ["gated_delta", "gated_delta_step", "w4_matvec", "w4_quantize"]

_L3 = ctypes.c_long * 3
_VP, _INT, _LONG = ctypes.c_void_p, ctypes.c_int, ctypes.c_long


class _GatedDeltaArgs(ctypes.Structure):
    _fields_ = [(n, _INT) for n in ("dtype", "gate_dtype", "batch", "frames", "k_heads", "v_heads", "k_dim", "v_dim")] \
        + [("scale", ctypes.c_float)] + [(n, _VP) for n in ("q", "k", "v", "g", "beta", "out")] \
        + [(n, _L3) for n in ("q_stride", "k_stride", "v_stride", "g_stride", "beta_stride", "out_stride")] \
        + [(n, _VP) for n in ("state_in", "state_out", "lengths", "active")]


class _W4MatvecArgs(ctypes.Structure):
    _fields_ = [(n, _INT) for n in ("dtype", "scale_dtype", "rows", "in_dim", "out_dim", "group")] \
        + [("x", _VP), ("x_stride", _LONG), ("codes", _VP), ("codes_pitch", _LONG), ("scales", _VP), ("scales_stride", _LONG),
           ("zeros", _VP), ("zeros_pitch", _LONG), ("bias", _VP), ("out", _VP), ("out_stride", _LONG)]


class _W4QuantizeArgs(ctypes.Structure):
    _fields_ = [(n, _INT) for n in ("dtype", "in_dim", "out_dim", "group")] \
        + [("weight", _VP), ("weight_stride", _LONG), ("codes", _VP), ("codes_pitch", _LONG), ("scales", _VP), ("scales_stride", _LONG),
           ("zeros", _VP), ("zeros_pitch", _LONG)]


# the same as bytes: packing them is several times faster than a Structure
_GATED_DELTA, _W4_MATVEC = struct.Struct("@8i f 6P 18l 4P"), struct.Struct("@6i P l P l P l P l P P l")


def _torch():
    import torch
    return torch


# A call's own time counts where a hop takes 3 us on the device: what it needs of torch and of the library is looked up once.
class _Env:
    def __init__(self):
        torch = _torch()
        from torch.autograd import forward_ad
        self.forward_ad = forward_ad
        self.torch, self.tensor, self.grad, self.empty = torch, torch.Tensor, torch.is_grad_enabled, torch.empty
        self.dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self.f32, self.u8, self.i32 = torch.float32, torch.uint8, torch.int32
        # the current stream's handle by device index, without a Stream object where torch offers that
        self.stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
        self.fns: dict = {}

    def fn(self, name: str):
        f = self.fns.get(name)
        if f is None:
            f = self.fns[name] = getattr(_backend.load_library(), name)
        return f


_the_env: Optional[_Env] = None


def _env() -> _Env:
    global _the_env
    if _the_env is None:
        _the_env = _Env()
    return _the_env


def _code(t, name: str) -> int:
    try:
        return _env().dtypes[t.dtype]
    except KeyError:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}") from None


def _checked(device, shape, dtype, name: str, t):
    """`t`, a tensor of this device, shape and type whose last dimension is contiguous."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.device.type != "cuda" or t.device != device:
        raise ValueError(f"{name} must be on {device if device.type == 'cuda' else 'a GPU'}, not on {t.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and this operator has no backward pass: call it under torch.no_grad()")
    return t


def _strides(env, device, index, shape, dtype, name: str, t):
    """The strides of `t` after `_checked`, whose messages it has where something does not fit."""
    if isinstance(t, env.tensor) and t.get_device() == index >= 0 and t.shape == shape and t.dtype is dtype:
        s = t.stride()
        if (s[-1] == 1 or shape[-1] <= 1) and not (t.requires_grad and env.grad()):
            return s
    return _checked(device, shape, dtype, name, t).stride()


def _gate_strides(env, device, index, shape, dtype, name: str, t):
    """The same for a gate: it has one value per head, no contiguous dimension is asked of it."""
    if isinstance(t, env.tensor) and t.get_device() == index >= 0 and t.shape == shape and t.dtype is dtype and not (t.requires_grad and env.grad()):
        return t.stride()
    return _checked(device, (*shape, 1), dtype, name, t[..., None] if isinstance(t, env.tensor) and t.dim() == 3 else t).stride()


def _forward_mode(env) -> bool:
    """Outside a forward-mode level, the usual case, no tensor has a tangent and none is looked at."""
    return getattr(env.forward_ad, "_current_level", 0) >= 0


def _no_tangents(env, **tensors) -> None:
    for name, t in tensors.items():
        if isinstance(t, env.tensor) and env.forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} carries a tangent, and this operator has no derivative: take forward_ad.unpack_dual({name}).primal")


def _packed(fields, *values) -> bytes:
    try:
        return fields.pack(*values)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"a size or the scale is out of range: {e}") from None


def _call(env, fn, index, args, *workspace) -> None:
    rc = env.fn(fn)(index, args, *workspace, env.stream(index))
    if rc:
        _backend._check(rc)


def _gated(fn, q, k, v, g, beta, state_in, state_out, lengths, active, scale, out):
    env = _env()
    if _forward_mode(env):
        _no_tangents(env, q=q, k=k, v=v, g=g, beta=beta, state=state_in, state_out=state_out, out=out)
    for name, t in (("q", q), ("v", v), ("g", g)):
        if not isinstance(t, env.tensor):
            raise ValueError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if q.dim() != 4 or v.dim() != 4 or g.dim() != 3:
        name, t, n = ("q", q, 4) if q.dim() != 4 else ("v", v, 4) if v.dim() != 4 else ("g", g, 3)
        raise ValueError(f"{name} must have {n} dimensions, got shape {list(t.shape)}")
    dev, index, dt, gt = q.device, q.get_device(), q.dtype, g.dtype
    qshape = q.shape
    B, T, Hk, Dk = qshape
    _, _, Hv, Dv = v.shape
    vshape = (B, T, Hv, Dv)
    code = _code(q, "q")
    if gt is not env.f32 and gt is not dt:
        raise ValueError(f"g and beta must be float32 or {dt}, got {gt}")
    qs, ks, vs = _strides(env, dev, index, qshape, dt, "q", q), _strides(env, dev, index, qshape, dt, "k", k), _strides(env, dev, index, vshape, dt, "v", v)
    gs, bs = _gate_strides(env, dev, index, (B, T, Hv), gt, "g", g), _gate_strides(env, dev, index, (B, T, Hv), gt, "beta", beta)
    for name, t in (("state", state_in), ("state_out", state_out)):
        if t is not None:
            _strides(env, dev, index, (B, Hv, Dk, Dv), env.f32, name, t)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        if state_out is state_in:
            break
    if lengths is not None:
        _strides(env, dev, index, (B,), env.i32, "lengths", lengths)
    if active is not None:
        _strides(env, dev, index, (B,), env.torch.bool if getattr(active, "dtype", None) == env.torch.bool else env.u8, "active", active)
    if out is None:
        # what the call leaves unwritten is 0 in a result of its own
        out = (env.empty if lengths is None and active is None else env.torch.zeros)(vshape, device=dev, dtype=dt)
        os = out.stride()
    else:
        os = _strides(env, dev, index, vshape, dt, "out", out)
    a = _packed(_GATED_DELTA, code, 0 if gt is env.f32 else code, B, T, Hk, Hv, Dk, Dv, 1.0 / math.sqrt(Dk) if scale is None else float(scale),
                q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(),
                *qs[:3], *ks[:3], *vs[:3], *gs[:3], *bs[:3], *os[:3], 0 if state_in is None else state_in.data_ptr(), 0 if state_out is None else state_out.data_ptr(),
                0 if lengths is None else lengths.data_ptr(), 0 if active is None else active.data_ptr())
    if fn == "dpdf_gated_delta_step":
        _call(env, fn, index, a)
    else:
        need = env.fn("dpdf_gated_delta_workspace")(index, a)
        room = env.empty(need, device=dev, dtype=env.u8) if need else None        # given back to torch when the call is queued: this stream's next users follow it
        _call(env, fn, index, a, room.data_ptr() if need else None, need)
    return out


def gated_delta(q: "torch.Tensor", k: "torch.Tensor", v: "torch.Tensor", g: "torch.Tensor", beta: "torch.Tensor", *,
                state: "Optional[torch.Tensor]" = None, lengths: "Optional[torch.Tensor]" = None, scale: Optional[float] = None,
                out: "Optional[torch.Tensor]" = None, state_out: "Optional[torch.Tensor]" = None) -> "Tuple[torch.Tensor, torch.Tensor]":
    """The gated delta rule over a batch of clips: (outputs, states after the last frames).

        S' = exp(g_t) S_{t-1};  e_t = beta_t (v_t - S'^T k_t);  S_t = S' + k_t e_t^T;  o_t = scale S_t^T q_t

    q, k [B, T, Hk, Dk], v [B, T, Hv, Dv] of one type, Dk at most 128, Hv a multiple of Hk (value head h reads key head h // (Hv // Hk));
    g (log of the decay, at most 0 in a stable layer; -inf resets the state) and beta [B, T, Hv], float32 or the type of q; scale: 1/sqrt(Dk).
    Any strides, the last dimension contiguous (g, beta: any).  state [B, Hv, Dk, Dv] float32, contiguous: the states to go on from (zeros).
    lengths [B] int32: frames of each clip; those behind are neither read nor written (0 in a result made here).
    out, state_out: where to write (state_out may be `state`)."""
    torch = _torch()
    if state_out is None and isinstance(q, torch.Tensor) and isinstance(v, torch.Tensor) and q.dim() == 4 and v.dim() == 4:
        state_out = torch.empty((q.shape[0], v.shape[2], q.shape[3], v.shape[3]), device=q.device, dtype=torch.float32)
    out = _gated("dpdf_gated_delta", q, k, v, g, beta, state, state_out, lengths, None, scale, out)
    return out, state_out


def gated_delta_step(q: "torch.Tensor", k: "torch.Tensor", v: "torch.Tensor", g: "torch.Tensor", beta: "torch.Tensor", state: "torch.Tensor", *,
                     active: "Optional[torch.Tensor]" = None, scale: Optional[float] = None,
                     out: "Optional[torch.Tensor]" = None) -> "torch.Tensor":
    """One hop, or a few, of live streams: `gated_delta` with one stream per row whose `state` is updated in place.

    active [S] uint8 or bool: the streams that have hops; rows of the others are neither read nor written (0 in a result made here), and
    their states stay as they are.  Everything else as in `gated_delta`; many frames are faster there."""
    if state is None:
        raise ValueError("a step needs its state")
    return _gated("dpdf_gated_delta_step", q, k, v, g, beta, state, state, None, active, scale, out)


def w4_matvec(x: "torch.Tensor", codes: "torch.Tensor", scales: "torch.Tensor", *, zeros: "Optional[torch.Tensor]" = None,
              bias: "Optional[torch.Tensor]" = None, group: int = 64, out: "Optional[torch.Tensor]" = None) -> "torch.Tensor":
    """A dense layer with 4-bit weights for a few rows: y[m, n] = sum_k x[m, k] (code[n, k] - zero[n, k // group]) scale[n, k // group] + bias[n].

    x [M, K] (or [K]); codes [N, (K + 1) // 2] uint8, weight 2 i in the lower half of byte i; scales [N, ceil(K / group)] float32 or the type
    of x; zeros [N, ceil(K / group)] uint8, 0 .. 15 (8 everywhere if not given); bias [N] of the type of x; group a multiple of 32, the last
    one may be short.  `w4_quantize` makes codes, scales and zeros."""
    env = _env()
    if _forward_mode(env):
        _no_tangents(env, x=x, scales=scales, bias=bias, out=out)
    for name, t in (("x", x), ("codes", codes), ("scales", scales)):
        if not isinstance(t, env.tensor):
            raise ValueError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if x.dim() not in (1, 2) or codes.dim() != 2:
        raise ValueError(f"x must be [M, K] or [K] and codes [N, (K + 1) // 2], got {list(x.shape)} and {list(codes.shape)}")
    xshape, dev, index, dt, st = x.shape, x.device, x.get_device(), x.dtype, scales.dtype
    M, K = xshape if len(xshape) == 2 else (1, xshape[0])
    N = codes.shape[0]
    yshape = (M, N) if len(xshape) == 2 else (N,)
    code, group = _code(x, "x"), int(group)
    if group < 32 or group % 32:
        raise ValueError(f"group must be a multiple of 32, got {group}")
    if st is not env.f32 and st is not dt:
        raise ValueError(f"scales must be float32 or {dt}, got {st}")
    groups = -(-K // group)
    xs, cs = _strides(env, dev, index, xshape, dt, "x", x), _strides(env, dev, index, (N, (K + 1) // 2), env.u8, "codes", codes)
    ss = _strides(env, dev, index, (N, groups), st, "scales", scales)
    zs = _strides(env, dev, index, (N, groups), env.u8, "zeros", zeros) if zeros is not None else (0,)
    if bias is not None:
        _strides(env, dev, index, (N,), dt, "bias", bias)
    if out is None:
        out = env.empty(yshape, device=dev, dtype=dt)
        ys = out.stride()
    else:
        ys = _strides(env, dev, index, yshape, dt, "out", out)
    _call(env, "dpdf_w4_matvec", index,
          _packed(_W4_MATVEC, code, 0 if st is env.f32 else code, M, K, N, group, x.data_ptr(), xs[0] if len(xshape) == 2 else K, codes.data_ptr(), cs[0],
                  scales.data_ptr(), ss[0], 0 if zeros is None else zeros.data_ptr(), zs[0], 0 if bias is None else bias.data_ptr(), out.data_ptr(), ys[0] if len(xshape) == 2 else N))
    return out


def w4_quantize(weight: "torch.Tensor", *, group: int = 64, symmetric: bool = False) -> "Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]":
    """(codes, scales, zeros) of a weight matrix [N, K] for `w4_matvec`; scales have the weight's type, zeros is None where symmetric.

    A group's range, 0 included, is divided into 15 steps (symmetric: its largest magnitude into 7); codes are the nearest, ties to even, under
    the scale as it is stored; a group with a weight that is not finite has the scale NaN.  Rows of codes start at multiples of 16 bytes, which is what `w4_matvec` reads fastest."""
    torch = _torch()
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be a torch tensor [N, K]")
    if _forward_mode(_env()):
        _no_tangents(_env(), weight=weight)
    code, group = _code(weight, "weight"), int(group)
    if group < 32 or group % 32:
        raise ValueError(f"group must be a multiple of 32, got {group}")
    dev, (N, K) = weight.device, weight.shape
    _checked(dev, (N, K), weight.dtype, "weight", weight.detach())
    groups = -(-K // group)
    pitch = -(-((K + 1) // 2) // 16) * 16
    codes = torch.empty((N, pitch), device=dev, dtype=torch.uint8)[:, :(K + 1) // 2]
    scales = torch.empty((N, groups), device=dev, dtype=weight.dtype)
    zeros = None if symmetric else torch.empty((N, groups), device=dev, dtype=torch.uint8)
    a = _W4QuantizeArgs(code, K, N, group, weight.data_ptr(), weight.stride(0), codes.data_ptr(), pitch, scales.data_ptr(), groups,
                        zeros.data_ptr() if zeros is not None else None, groups)
    _call(_env(), "dpdf_w4_quantize", dev.index, ctypes.addressof(a))
    return codes, scales, zeros
