"""Stand-alone operators on device tensors: the gated delta rule (a recurrence over frames with a matrix state) over whole clips and hop by
hop, and dense layers with 4-bit weights for a few rows -- the parts of a recurrent layer beside the engine's own (`dpdf_gated_delta`,
`dpdf_gated_delta_step`, `dpdf_w4_matvec`, `dpdf_w4_quantize` of include/dpdfnet_hip.h).

Tensors are torch tensors on one HIP device, float32, float16 or bfloat16; calls are queued on torch's current stream of that device,
allocate nothing beside their results (and, for a few long clips, a workspace) through torch and wait for nothing, so they can be captured into a graph.  Sums, states and accumulators are fp32
whatever the tensors' type.  There is no backward pass: tensors that require a gradient are refused while gradients are recorded.  Wrong
types, shapes and overlaps raise ValueError, failures of the device RuntimeError."""
from __future__ import annotations

import ctypes
import math
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


def _torch():
    import torch
    return torch


_dtypes = None


def _code(t, name: str) -> int:
    global _dtypes
    if _dtypes is None:
        torch = _torch()
        _dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    try:
        return _dtypes[t.dtype]
    except KeyError:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}") from None


def _checked(device, shape, dtype, name: str, t):
    """`t`, a tensor of this device, shape (None: any) and type whose last dimension is contiguous."""
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


def _call(fn, device, args, *workspace) -> None:
    stream = _torch().cuda.current_stream(device).cuda_stream
    _backend._check(getattr(_backend.load_library(), fn)(device.index, ctypes.addressof(args), *workspace, stream))


def _gated(fn, q, k, v, g, beta, state_in, state_out, lengths, active, scale, out):
    torch = _torch()
    for name, t in (("q", q), ("v", v), ("g", g)):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a torch tensor, got {type(t).__name__}")
        if t.dim() != (3 if name == "g" else 4):
            raise ValueError(f"{name} must have {3 if name == 'g' else 4} dimensions, got shape {list(t.shape)}")
    dev, dt = q.device, q.dtype
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    code = _code(q, "q")
    if g.dtype != torch.float32 and g.dtype != dt:
        raise ValueError(f"g and beta must be float32 or {dt}, got {g.dtype}")
    _checked(dev, (B, T, Hk, Dk), dt, "q", q)
    _checked(dev, (B, T, Hk, Dk), dt, "k", k)
    _checked(dev, (B, T, Hv, Dv), dt, "v", v)
    # gates have one value per head: no contiguous dimension is asked of them
    for name, t in (("g", g), ("beta", beta)):
        _checked(dev, (B, T, Hv, 1), g.dtype, name, t[..., None] if isinstance(t, torch.Tensor) and t.dim() == 3 else t)
    for name, t in (("state", state_in), ("state_out", state_out)):
        if t is not None and not _checked(dev, (B, Hv, Dk, Dv), torch.float32, name, t).is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if lengths is not None:
        _checked(dev, (B,), torch.int32, "lengths", lengths)
    if active is not None:
        _checked(dev, (B,), torch.bool if getattr(active, "dtype", None) == torch.bool else torch.uint8, "active", active)
    if out is None:
        # what the call leaves unwritten is 0 in a result of its own
        out = (torch.empty if lengths is None and active is None else torch.zeros)((B, T, Hv, Dv), device=dev, dtype=dt)
    else:
        _checked(dev, (B, T, Hv, Dv), dt, "out", out)
    a = _GatedDeltaArgs(code, 0 if g.dtype == torch.float32 else code, B, T, Hk, Hv, Dk, Dv, 1.0 / math.sqrt(Dk) if scale is None else scale,
                        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(),
                        q.stride()[:3], k.stride()[:3], v.stride()[:3], g.stride(), beta.stride(), out.stride()[:3],
                        state_in.data_ptr() if state_in is not None else None, state_out.data_ptr() if state_out is not None else None,
                        lengths.data_ptr() if lengths is not None else None, active.data_ptr() if active is not None else None)
    if fn == "dpdf_gated_delta_step":
        _call(fn, dev, a)
    else:
        need = _backend.load_library().dpdf_gated_delta_workspace(dev.index, ctypes.addressof(a))
        room = torch.empty(need, device=dev, dtype=torch.uint8) if need else None        # given back to torch when the call is queued: this stream's next users follow it
        _call(fn, dev, a, room.data_ptr() if need else None, need)
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
    torch = _torch()
    for name, t in (("x", x), ("codes", codes), ("scales", scales)):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if x.dim() not in (1, 2) or codes.dim() != 2:
        raise ValueError(f"x must be [M, K] or [K] and codes [N, (K + 1) // 2], got {list(x.shape)} and {list(codes.shape)}")
    x2 = x if x.dim() == 2 else x[None]
    dev, dt = x.device, x.dtype
    M, K = x2.shape
    N = codes.shape[0]
    code, group = _code(x, "x"), int(group)
    if group < 32 or group % 32:
        raise ValueError(f"group must be a multiple of 32, got {group}")
    if scales.dtype != torch.float32 and scales.dtype != dt:
        raise ValueError(f"scales must be float32 or {dt}, got {scales.dtype}")
    groups = -(-K // group)
    _checked(dev, (M, K), dt, "x", x2)
    _checked(dev, (N, (K + 1) // 2), torch.uint8, "codes", codes)
    _checked(dev, (N, groups), scales.dtype, "scales", scales)
    if zeros is not None:
        _checked(dev, (N, groups), torch.uint8, "zeros", zeros)
    if bias is not None:
        _checked(dev, (N,), dt, "bias", bias)
    if out is None:
        out = torch.empty((M, N) if x.dim() == 2 else (N,), device=dev, dtype=dt)
    else:
        _checked(dev, (M, N) if x.dim() == 2 else (N,), dt, "out", out)
    a = _W4MatvecArgs(code, 0 if scales.dtype == torch.float32 else code, M, K, N, group, x.data_ptr(), x2.stride(0), codes.data_ptr(), codes.stride(0),
                      scales.data_ptr(), scales.stride(0), zeros.data_ptr() if zeros is not None else None, zeros.stride(0) if zeros is not None else 0,
                      bias.data_ptr() if bias is not None else None, out.data_ptr(), out.stride(0) if out.dim() == 2 else N)
    _call("dpdf_w4_matvec", dev, a)
    return out


def w4_quantize(weight: "torch.Tensor", *, group: int = 64, symmetric: bool = False) -> "Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]":
    """(codes, scales, zeros) of a weight matrix [N, K] for `w4_matvec`; scales have the weight's type, zeros is None where symmetric.

    A group's range, 0 included, is divided into 15 steps (symmetric: its largest magnitude into 7); codes are the nearest, ties to even, under
    the scale as it is stored.  Rows of codes start at multiples of 16 bytes, which is what `w4_matvec` reads fastest."""
    torch = _torch()
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be a torch tensor [N, K]")
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
    _call("dpdf_w4_quantize", dev, a)
    return codes, scales, zeros
