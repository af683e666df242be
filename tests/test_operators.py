"""The stand-alone operators (`dpdfnet_amd.operators`): gated delta rule over clips and hop by hop, dense layers with 4-bit weights.
CPU: refusals, argument layouts, the alias.  GPU: every form against its definition in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32.  A frame of the recurrence takes sums of Dk products and a chunk sums of 64 more; with |k| <= 1 and
0 <= beta <= 1 a frame's error is not amplified later, so after T frames at most T (Dk + 64) roundings of relative size u have added up,
like a random walk: TOL = 8 deviations = 8 sqrt(T (Dk + 64)) u of the largest magnitude.  On top comes the result's own rounding, half a step of
its type relative to the value (bf16 2^-8, fp16 2^-11)."""
import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from dpdfnet_amd import backend, operators

ROOT = Path(__file__).resolve().parents[1]
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------------------------------------------------------------------
# definitions in 64 bits, on the CPU
# ---------------------------------------------------------------------------------------------------------------------------------------
def delta_rule(q, k, v, g, beta, state=None, lengths=None, scale=None):
    q, k, v, g, beta = (t.detach().double().cpu() for t in (q, k, v, g, beta))
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    head = torch.arange(Hv) // (Hv // Hk)
    q, k = q[:, :, head], k[:, :, head]
    scale = 1 / math.sqrt(Dk) if scale is None else scale
    S = torch.zeros(B, Hv, Dk, Dv, dtype=torch.float64) if state is None else state.detach().double().cpu().clone()
    out = torch.zeros(B, T, Hv, Dv, dtype=torch.float64)
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long()
    for t in range(T):
        on = (t < n)[:, None, None]
        Sd = S * g[:, t].exp()[..., None, None]
        e = beta[:, t, :, None] * (v[:, t] - (Sd * k[:, t, :, :, None]).sum(2))
        new = Sd + k[:, t, :, :, None] * e[:, :, None]
        out[:, t] = torch.where(on, scale * (new * q[:, t, :, :, None]).sum(2), out[:, t])
        S = torch.where(on[..., None], new, S)
    return out, S


def w4_layer(x, codes, scales, zeros, bias, group):
    x, codes, scales = x.detach().double().cpu(), codes.cpu(), scales.double().cpu()
    K = x.shape[-1]
    k = torch.arange(K)
    c = ((codes[:, k // 2].int() >> (4 * (k % 2))) & 15).double()
    z = 8.0 if zeros is None else zeros.cpu().double()[:, k // group]
    w = (c - z) * scales[:, k // group]
    y = x @ w.t()
    return (y if bias is None else y + bias.double().cpu()), x.abs() @ w.abs().t()


def inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=0, device="cuda", g_std=1.0):
    gen = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=gen)
    q, k = (torch.nn.functional.normalize(r(B, T, Hk, Dk), dim=-1).to(dtype) for _ in range(2))
    g = -torch.rand(B, T, Hv, generator=gen) * torch.exp(g_std * r(Hv) - 2)
    return [t.to(device) for t in (q, k, r(B, T, Hv, Dv).to(dtype), g, torch.sigmoid(r(B, T, Hv)))]


def tol(T, Dk):
    return 8 * math.sqrt(T * (Dk + 64)) * U


def near(got, ref, rel, half_step=0.0, tiny=0.0):
    """|got - ref| <= rel * (largest |ref|) + half a step of the result's type."""
    got = got.detach().double().cpu()
    assert got.shape == ref.shape
    top = float(ref.abs().max()) if ref.numel() else 0.0
    bound = rel * top + half_step * ref.abs() * (1 + rel) + tiny
    off = (got - ref).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= bound).all()), f"worst {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


# ---------------------------------------------------------------------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------------------------------------------------------------------
def test_argument_structures_match_the_header(tmp_path):
    pairs = {"dpdf_gated_delta_args": operators._GatedDeltaArgs, "dpdf_w4_matvec_args": operators._W4MatvecArgs, "dpdf_w4_quantize_args": operators._W4QuantizeArgs}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "dpdfnet_hip.h"\nint main(void) {\n'
    for name, cls in pairs.items():
        src += f'printf("{name} %zu", sizeof({name}));' + "".join(f'printf(" %zu", offsetof({name}, {f[0]}));' for f in cls._fields_) + 'printf("\\n");\n'
    (tmp_path / "s.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-I" + str(ROOT / "include"), "-o", str(tmp_path / "s"), str(tmp_path / "s.c")], check=True)
    for line in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, *nums = line.split()
        cls = pairs[name]
        assert [int(n) for n in nums] == [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]


@pytest.mark.parametrize("fields, cls", [(operators._GATED_DELTA, operators._GatedDeltaArgs), (operators._W4_MATVEC, operators._W4MatvecArgs)])
def test_packed_arguments_are_the_structures(fields, cls):
    flat = [n for n, t in cls._fields_ for _ in range(3 if t is operators._L3 else 1)]
    a = cls.from_buffer_copy(fields.pack(*(i + 1 for i in range(len(flat)))))
    got = []
    for n, t in cls._fields_:
        got += list(getattr(a, n)) if t is operators._L3 else [getattr(a, n)]
    assert got == [i + 1 for i in range(len(flat))]
    with pytest.raises(ValueError, match="out of range"):
        operators._packed(fields, *(2 ** 40 for _ in flat))


def test_operators_are_reachable_under_both_names():
    import dpdfnet.operators as alias
    assert alias is operators
    assert set(operators.__all__) == {"gated_delta", "gated_delta_step", "w4_matvec", "w4_quantize"}


def _c_gated(step=False, workspace=None, **change):
    """A call of the C entry on made-up addresses with one thing changed: refused before any of them is looked at."""
    B, T, Hk, Hv, Dk, Dv = 2, 3, 2, 4, 16, 8
    v = dict(dtype=2, gate_dtype=0, batch=B, frames=T, k_heads=Hk, v_heads=Hv, k_dim=Dk, v_dim=Dv, scale=1.0,
             q=0x1000000, k=0x2000000, v=0x3000000, g=0x4000000, beta=0x5000000, out=0x6000000,
             q_stride=(T * Hk * Dk, Hk * Dk, Dk), k_stride=(T * Hk * Dk, Hk * Dk, Dk), v_stride=(T * Hv * Dv, Hv * Dv, Dv),
             g_stride=(T * Hv, Hv, 1), beta_stride=(T * Hv, Hv, 1), out_stride=(T * Hv * Dv, Hv * Dv, Dv),
             state_in=0x7000000, state_out=0x7000000, lengths=None, active=None)
    v.update(change)
    a = operators._GatedDeltaArgs(*[v[f[0]] for f in operators._GatedDeltaArgs._fields_])
    L = backend.load_library()
    rc = L.dpdf_gated_delta_step(0, ctypes.addressof(a), None) if step else L.dpdf_gated_delta(0, ctypes.addressof(a), workspace, 1 << 20, None)
    return rc, L.dpdf_last_error().decode()


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "dtypes"), (dict(dtype=-1), "dtypes"), (dict(gate_dtype=1), "dtypes"), (dict(batch=-1), "negative"), (dict(frames=-1), "negative"),
    (dict(k_heads=3), "multiple"), (dict(k_heads=0), "multiple"), (dict(v_heads=0), "multiple"), (dict(k_dim=0), "head sizes"), (dict(k_dim=129), "head sizes"),
    (dict(v_dim=0), "head sizes"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(v=0x3000001), "aligned"), (dict(g=0x4000002), "aligned"), (dict(state_in=0x7000002, state_out=None), "aligned"), (dict(lengths=0x8000001), "aligned"),
    (dict(q_stride=(-1, 1, 1)), "negative stride"), (dict(out_stride=(0, 32, 8)), "share"), (dict(out_stride=(96, 32, 7)), "share"), (dict(out_stride=(96, 24, 8)), "share"),
    (dict(out=0x3000000), "overlaps an input"), (dict(out=0x1000000 - 2), "overlaps an input"), (dict(out=0x7000000), "out overlaps"),
    (dict(state_out=0x7000004), "in part"), (dict(state_out=0x2000000), "overlaps an input"), (dict(active=0x9000000), "mask"),
    (dict(batch=1 << 30), "too large"), (dict(frames=(1 << 30) + 1), "too large"), (dict(workspace=0x9000008), "aligned"),
 (dict(k=1 << 45, k_stride=(1 << 38, 1 << 30, 16)), "frame to frame"), (dict(out=1 << 45, out_stride=(1 << 40, 1 << 31, 8)), "frame to frame"),
    (dict(frames=2, out=1 << 45, out_stride=(1 << 40, 1 << 25, 8)), "frame to frame"), (dict(frames=2, v=1 << 45, v_stride=(1 << 40, 1 << 24, 8)), "frame to frame"),
])
def test_gated_delta_refusals(change, word):
    rc, msg = _c_gated(**change)
    assert rc == -1 and word in msg, (rc, msg)


def test_gated_delta_step_refusals_and_empty_calls():
    one = dict(batch=1, frames=1, k_heads=1, v_heads=1, k_dim=128, state_in=1 << 50, state_out=1 << 50, v=1 << 51, out=1 << 52)
    for n in ("q", "k", "v", "g", "beta", "out"):
        one[n + "_stride"] = (1 << 22,) * 3
    rc, msg = _c_gated(step=True, v_dim=1 << 22, **one)
    assert rc == -1 and "128 x 4194304 is too large" in msg, (rc, msg)
    assert _c_gated(step=True, lengths=0x8000000)[0] == -1
    assert _c_gated(step=True, state_in=None)[0] == -1 and _c_gated(step=True, state_out=None)[0] == -1
    L = backend.load_library()
    assert L.dpdf_gated_delta(0, None, None, 0, None) == -1 and L.dpdf_gated_delta_workspace(0, None) == 0 and L.dpdf_gated_delta_step(0, None, None) == -1
    assert L.dpdf_w4_matvec(0, None, None) == -1 and L.dpdf_w4_quantize(0, None, None) == -1
    # nothing to do: no device is touched
    assert _c_gated(batch=0)[0] == 0 and _c_gated(step=True, batch=0)[0] == 0 and _c_gated(step=True, frames=0)[0] == 0
    assert _c_gated(frames=0, state_out=None)[0] == 0
    if backend.device_count() == 0:
        assert _c_gated(frames=0)[0] == -2                                 # the states are still to be written
        assert _c_gated()[0] == -2 and _c_gated(step=True)[0] == -2        # no GPU: a failure, nothing computed elsewhere


@pytest.mark.parametrize("change", [
    dict(lengths=0x6000000), dict(lengths=0x6000000 - 4), dict(lengths=0x7000000), dict(lengths=0x7000000 + 2 * 4 * 16 * 8 * 4 - 4), dict(frames=0, lengths=0x7000000),
    dict(step=True, active=0x6000001), dict(step=True, active=0x7000000 + 2 * 4 * 16 * 8 * 4 - 1), dict(step=True, active=0x7000000 - 1),
])
def test_lengths_and_masks_in_an_outputs_memory_are_refused(change):
    rc, msg = _c_gated(**change)
    assert rc == -1 and "overlaps an input" in msg, (rc, msg)


def test_sizes_next_to_what_32_bits_count_are_refused():
    big = (1 << 30) + 1
    for change in (dict(in_dim=big), dict(out_dim=big), dict(in_dim=(1 << 31) - 1), dict(out_dim=(1 << 31) - 1, out_stride=(1 << 31) - 1)):
        change = dict(x=1 << 44, x_stride=1 << 32, codes=2 << 44, codes_pitch=1 << 31, scales=3 << 44, scales_stride=1 << 27, zeros=4 << 44, zeros_pitch=1 << 27, bias=5 << 44,
                      out=6 << 44, out_stride=big) | change
        rc, msg = _c_w4(**change)
        assert rc == -1 and "too large" in msg, (rc, msg)
    a = operators._W4QuantizeArgs(0, (1 << 31) - 1, 1, 32, 1 << 44, 1 << 31, 2 << 44, 1 << 31, 3 << 44, 1 << 27, None, 0)
    L = backend.load_library()
    assert L.dpdf_w4_quantize(0, ctypes.addressof(a), None) == -1 and "too large" in L.dpdf_last_error().decode()
    rc, msg = _c_gated(frames=0, batch=1, k_heads=1, v_heads=1, k_dim=1, v_dim=(1 << 31) - 1, state_in=1 << 44, state_out=2 << 44)
    assert rc == -1 and "head sizes" in msg, (rc, msg)


def test_calls_of_more_threads_than_a_launch_has_are_refused():
    """2^32 threads: 2^26 heads of a step's one wave, 2^24 of a clip's four, tiles of up to eight waves; one less of them is no such case."""
    far = {n: (i + 1) << 44 for i, n in enumerate(("q", "k", "v", "g", "beta", "out"))}
    far.update({n + "_stride": (1, 1, 1) for n in far}, frames=1, k_heads=1, v_heads=1, k_dim=1, v_dim=1, state_in=8 << 44, state_out=8 << 44)
    ok = 0 if backend.device_count() else -2
    for step, most in ((True, 1 << 26), (False, 1 << 24)):
        rc, msg = _c_gated(step=step, **{**far, "batch": most})
        assert rc == -1 and "too large for one call" in msg, (rc, msg)
        if ok:                                                                # where no device is there, what is not refused ends at that
            assert _c_gated(step=step, **{**far, "batch": most - 1})[0] == ok
    w4 = dict(in_dim=1024, x=1 << 44, x_stride=1024, codes=2 << 44, codes_pitch=512, scales=3 << 44, zeros=4 << 44, bias=5 << 44, out=6 << 44, out_dim=1 << 20, out_stride=1 << 20, scales_stride=32, zeros_pitch=32)
    rc, msg = _c_w4(rows=1 << 14, **w4)                                       # 2^26 tiles, four to a workgroup of four waves
    assert rc == -1 and "too many for one call" in msg, (rc, msg)
    if ok:
        assert _c_w4(rows=(1 << 14) - 16, **w4)[0] == ok


def _c_w4(**change):
    v = dict(dtype=1, scale_dtype=1, rows=2, in_dim=100, out_dim=6, group=32, x=0x1000000, x_stride=100, codes=0x2000000, codes_pitch=50,
             scales=0x3000000, scales_stride=4, zeros=0x4000000, zeros_pitch=4, bias=0x5000000, out=0x6000000, out_stride=6)
    v.update(change)
    a = operators._W4MatvecArgs(*[v[f[0]] for f in operators._W4MatvecArgs._fields_])
    L = backend.load_library()
    return L.dpdf_w4_matvec(0, ctypes.addressof(a), None), L.dpdf_last_error().decode()


@pytest.mark.parametrize("change, word", [
    (dict(dtype=9), "dtype"), (dict(scale_dtype=2), "dtypes"), (dict(rows=-1), "negative"), (dict(in_dim=0), "empty"), (dict(out_dim=0), "empty"),
    (dict(group=0), "group"), (dict(group=48), "group"), (dict(group=-32), "group"), (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"),
    (dict(out=None), "null"), (dict(x_stride=-1), "negative stride"), (dict(out_stride=5), "share"), (dict(x=0x1000001), "aligned"), (dict(scales=0x3000001), "aligned"),
    (dict(out=0x1000000), "overlaps"), (dict(out=0x2000020), "overlaps"), (dict(out=0x3000000), "overlaps"), (dict(out=0x4000000), "overlaps"), (dict(out=0x5000002), "overlaps"),
])
def test_w4_refusals(change, word):
    rc, msg = _c_w4(**change)
    assert rc == -1 and word in msg, (rc, msg)


def test_w4_empty_call_and_quantize_refusals():
    assert _c_w4(rows=0)[0] == 0
    base = dict(dtype=0, in_dim=100, out_dim=6, group=32, weight=0x1000000, weight_stride=100, codes=0x2000000, codes_pitch=50,
                scales=0x3000000, scales_stride=4, zeros=0x4000000, zeros_pitch=4)
    L = backend.load_library()
    for change in (dict(dtype=5), dict(in_dim=0), dict(group=16), dict(weight=None), dict(codes=None), dict(scales=None), dict(codes_pitch=49), dict(scales_stride=3),
                   dict(zeros_pitch=3), dict(weight_stride=-1), dict(weight=0x1000002), dict(scales=0x1000004), dict(codes=0x3000000), dict(zeros=0x2000010)):
        v = {**base, **change}
        a = operators._W4QuantizeArgs(*[v[f[0]] for f in operators._W4QuantizeArgs._fields_])
        assert L.dpdf_w4_quantize(0, ctypes.addressof(a), None) == -1, change


def test_python_layer_refuses_what_is_on_the_cpu_or_of_a_wrong_kind():
    q, k, v, g, beta = inputs(1, 2, 1, 2, 16, 16, F32, device="cpu")
    state = torch.zeros(1, 2, 16, 16)
    with pytest.raises(ValueError, match="GPU"):
        operators.gated_delta(q, k, v, g, beta)
    with pytest.raises(ValueError, match="GPU"):
        operators.gated_delta_step(q, k, v, g, beta, state)
    with pytest.raises(ValueError, match="state"):
        operators.gated_delta_step(q, k, v, g, beta, None)
    with pytest.raises(ValueError, match="tensor"):
        operators.gated_delta([1.0], k, v, g, beta)
    with pytest.raises(ValueError, match="dimensions"):
        operators.gated_delta(q[0], k, v, g, beta)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        operators.gated_delta(q.double(), k, v, g, beta)
    with pytest.raises(ValueError, match="GPU"):
        operators.w4_matvec(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1))
    with pytest.raises(ValueError, match="group"):
        operators.w4_matvec(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1), group=40)
    with pytest.raises(ValueError, match="GPU"):
        operators.w4_quantize(torch.zeros(4, 64))


def test_tangents_are_refused_before_anything_else():
    from torch.autograd import forward_ad
    q, k, v, g, beta = inputs(1, 2, 1, 2, 16, 16, F32, device="cpu")
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="v carries a tangent"):
            operators.gated_delta(q, k, forward_ad.make_dual(v, v), g, beta)
        with pytest.raises(ValueError, match="weight carries a tangent"):
            operators.w4_quantize(forward_ad.make_dual(torch.zeros(4, 64), torch.ones(4, 64)))
        with pytest.raises(ValueError, match="GPU"):
            operators.gated_delta(q, k, v, g, beta)


# ---------------------------------------------------------------------------------------------------------------------------------------
# GPU: the gated delta rule
# ---------------------------------------------------------------------------------------------------------------------------------------
CLIPS = [  # B, T, Hk, Hv, Dk, Dv
    (1, 1, 1, 1, 16, 16), (2, 2, 1, 1, 1, 1), (1, 16, 1, 2, 17, 33), (2, 63, 2, 2, 32, 16), (1, 64, 1, 3, 64, 64), (3, 65, 2, 4, 64, 48),
    (1, 127, 1, 1, 128, 128), (2, 130, 3, 3, 48, 100), (1, 257, 2, 6, 80, 17), (1, 400, 1, 2, 128, 64), (5, 70, 1, 1, 5, 130),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", CLIPS)
def test_clips_against_the_definition(shape, dtype):
    B, T, Hk, Hv, Dk, Dv = shape
    x = inputs(*shape, dtype, seed=T)
    state = 0.5 * torch.randn(B, Hv, Dk, Dv, generator=torch.Generator().manual_seed(1)).cuda()
    for s in (None, state):
        out, end = operators.gated_delta(*x, state=s)
        ref, rend = delta_rule(*x, state=s)
        near(out, ref, tol(T, Dk), HALF_STEP[dtype], TINY[dtype])
        near(end, rend, tol(T, Dk))
    assert torch.equal(state, 0.5 * torch.randn(B, Hv, Dk, Dv, generator=torch.Generator().manual_seed(1)).cuda())        # read only


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 16, 16), (2, 3, 1, 2, 1, 1), (3, 1, 2, 6, 17, 33), (4, 2, 1, 1, 64, 64), (2, 4, 2, 4, 128, 128), (1, 5, 1, 2, 100, 30),
                                   (7, 1, 4, 4, 48, 40)])
def test_steps_against_the_definition(shape, dtype):
    B, T, Hk, Hv, Dk, Dv = shape
    x = inputs(*shape, dtype, seed=B)
    state = 0.5 * torch.randn(B, Hv, Dk, Dv, generator=torch.Generator().manual_seed(1)).cuda()
    ref, rend = delta_rule(*x, state=state)
    ptr = state.data_ptr()
    out = operators.gated_delta_step(*x, state)
    assert state.data_ptr() == ptr
    near(out, ref, tol(T, Dk), HALF_STEP[dtype], TINY[dtype])
    near(state, rend, tol(T, Dk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Dk", [8, 16, 13, 24, 31, 40, 63, 72, 96, 95, 104, 128, 127])
def test_steps_of_every_size(Dk, dtype):
    x = inputs(2, 3, 1, 2, Dk, 36, dtype, seed=Dk)
    state = 0.5 * torch.randn(2, 2, Dk, 36, generator=torch.Generator().manual_seed(1)).cuda()
    ref, rend = delta_rule(*x, state=state)
    out = operators.gated_delta_step(*x, state)
    near(out, ref, tol(3, Dk), HALF_STEP[dtype], TINY[dtype])
    near(state, rend, tol(3, Dk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S, T, Hk, Hv, Dk, Dv", [(3, 4, 1, 2, 96, 40), (2, 3, 2, 2, 80, 100), (5, 2, 1, 1, 72, 3), (2, 5, 1, 3, 67, 33), (1, 6, 2, 4, 88, 16), (2, 2, 1, 1, 20, 36), (3, 3, 1, 1, 8, 1)])
def test_steps_of_sizes_between(S, T, Hk, Hv, Dk, Dv, dtype):
    x = inputs(S, T, Hk, Hv, Dk, Dv, dtype, seed=Dk + Dv)
    room = torch.full((S * Hv * Dk * Dv + 64,), math.nan, device="cuda")                # nothing beside the state is taken for it or written
    state = room[32:-32].view(S, Hv, Dk, Dv)
    state.copy_(0.5 * torch.randn(S, Hv, Dk, Dv, generator=torch.Generator().manual_seed(1)))
    ref, rend = delta_rule(*x, state=state)
    wide = torch.full((S, T, Hv, Dv + 5), 3.0, dtype=dtype, device="cuda")
    out = operators.gated_delta_step(*x, state, out=wide[..., 2:Dv + 2])
    near(out, ref, tol(T, Dk), HALF_STEP[dtype], TINY[dtype])
    near(state, rend, tol(T, Dk))
    assert bool(room[:32].isnan().all()) and bool(room[-32:].isnan().all())
    assert bool((wide[..., :2] == 3).all()) and bool((wide[..., Dv + 2:] == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gates_of_the_values_type(dtype):
    x = inputs(2, 100, 2, 2, 32, 32, dtype, seed=4)
    x[3], x[4] = x[3].to(dtype), x[4].to(dtype)
    out, end = operators.gated_delta(*x)
    ref, rend = delta_rule(*x)
    near(out, ref, tol(100, 32), HALF_STEP[dtype], TINY[dtype])
    near(end, rend, tol(100, 32))
    state = torch.zeros(2, 2, 32, 32, device="cuda")
    out = operators.gated_delta_step(*[t[:, :3] for t in x], state)
    ref, rend = delta_rule(*[t[:, :3] for t in x])
    near(out, ref, tol(3, 32), HALF_STEP[dtype], TINY[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("drop, up", [(-140.0, 43.0), (-200.0, 75.0)])
def test_growth_behind_a_reset_brings_nothing_back(drop, up, dtype):
    """g = -inf empties the state whatever follows; a large negative g and growth after it are what their sum is.  Without writes (beta = 0) the
    outputs are exp(sum of g) S0^T q: 0 behind the reset, exp(-140 + 86) of it for the second head.  exp's argument, -78 in powers of two, is off by
    half a step of fp32 there (2^-18), the result by as much, the sums by tol().  Growth by 150 in two frames is more than fp32
    holds: from the second of them on clips give NaN, and everything before is as it was."""
    T, D, scale = 40, 32, 1e20 if dtype != F16 else 1.0
    q, k, v, g, beta = inputs(1, T, 1, 3, D, D, dtype, seed=31)
    g, beta = torch.zeros_like(g), torch.zeros_like(beta)
    for h, down in enumerate((-math.inf, drop, -1000.0)):
        g[:, 3, h], g[:, 5:7, h] = down, up
    state = torch.randn(1, 3, D, D, generator=torch.Generator().manual_seed(1)).cuda()
    out, end = operators.gated_delta(q, k, v, g, beta, state=state, scale=scale)
    ref, rend = delta_rule(q, k, v, g, beta, state=state, scale=scale)
    n = 6 if 2 * up > 88 else T
    near(out[:, :3], ref[:, :3], tol(T, D), HALF_STEP[dtype], TINY[dtype])
    assert bool((out[:, 3:n, [0, 2]] == 0).all())
    if n < T:
        assert bool(out[:, n:].isnan().all()) and bool(end.isnan().all())
    else:
        assert bool((end[:, [0, 2]] == 0).all())
        near(out[:, 7:, 1], ref[:, 7:, 1], tol(T, D) + 2.0 ** -16, HALF_STEP[dtype], TINY[dtype])
        near(end[:, 1], rend[:, 1], tol(T, D) + 2.0 ** -16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T, at", [(90, 20), (90, 70), (1200, 700)])
def test_growth_beyond_fp32_spares_what_is_before_it(T, at, dtype):
    """exp(g) of one frame, or of several together, outside fp32: NaN from there on, the frames before bit for bit, and the other head."""
    x = inputs(1, T, 1, 2, 32, 32, dtype, seed=T)
    clean, cend = operators.gated_delta(*x)
    for grow in ([100.0], [40.0, 40.0, 40.0]):
        g, first = x[3].clone(), at + 1 - len(grow)
        g[0, first:at + 1, 0] = torch.tensor(grow, device="cuda")
        out, end = operators.gated_delta(*x[:3], g, x[4])
        assert torch.equal(out[:, :first], clean[:, :first]) and torch.equal(out[:, :, 1], clean[:, :, 1]) and torch.equal(end[:, 1], cend[:, 1])
        assert dtype == F16 or bool(out[:, :at, 0].isfinite().all())              # exp(80) is in range, but not of fp16
        assert bool(out[:, at:, 0].isnan().all()) and bool(end[:, 0].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_hard_gates_and_keys(dtype, D):
    """No decay, decays that empty the state within a frame, resets by -inf, beta of 0 and 1, and one key in every frame."""
    T = 150
    q, k, v, g, beta = inputs(1, T, 1, 6, D, 32, dtype, seed=9)
    g = g.clone()
    g[:, :, 0] = 0
    g[:, :, 1] = -30
    g[:, ::37, 2] = -math.inf
    g[:, :, 3] = torch.where(torch.rand(1, T, generator=torch.Generator().manual_seed(2)).cuda() < 0.5, -100.0, -0.001)
    beta = beta.clone()
    beta[:, ::2, 4] = 0
    beta[:, :, 0] = 1
    for keys in (k, k[:, :1].expand(-1, T, -1, -1), torch.zeros_like(k)):
        out, end = operators.gated_delta(q, keys, v, g, beta)
        ref, rend = delta_rule(q, keys, v, g, beta)
        near(out, ref, tol(T, D), HALF_STEP[dtype], TINY[dtype])
        near(end, rend, tol(T, D))
        state = torch.zeros(1, 6, D, 32, device="cuda")
        out = operators.gated_delta_step(q[:, :40], keys[:, :40], v[:, :40], g[:, :40], beta[:, :40], state)
        near(out, ref[:, :40], tol(40, D), HALF_STEP[dtype], TINY[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [(0, 0, 0), (1, 64, 0), (65, 130, 3), (130, 129, 128), (-5, 1000, 66)])
def test_ragged_clips_leave_the_rest_alone(lens):
    B, T, dtype = 3, 130, BF16
    x = inputs(B, T, 1, 2, 32, 48, dtype, seed=3)
    held = torch.tensor([min(max(n, 0), T) for n in lens])
    for b in range(B):                        # nothing behind the end may be looked at
        for t in x:
            t[b, held[b]:] = math.nan
    state = torch.randn(B, 2, 32, 48, generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.full((B, T, 2, 48), 7.0, device="cuda", dtype=dtype)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got, end = operators.gated_delta(*x, state=state, lengths=lengths, out=out)
    assert got is out
    ref, rend = delta_rule(*[torch.nan_to_num(t, nan=0.0) for t in x], state=state, lengths=held)
    on = (torch.arange(T)[None] < held[:, None])[..., None, None].expand_as(ref)
    assert bool((out.cpu()[~on] == 7.0).all())
    if bool(on.any()):
        near(torch.where(on, out.cpu().double(), 0.0), ref, tol(T, 32), HALF_STEP[dtype], TINY[dtype])
    near(end, rend, tol(T, 32))
    for b in range(B):
        if held[b] == 0:
            assert torch.equal(end[b], state[b])
    assert bool((operators.gated_delta(*x, lengths=lengths)[0].cpu()[~on] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B, T, lens, D", [(256, 40, "any", 48), (200, 70, "any", 64), (180, 33, "equal", 48), (257, 20, "any", 48), (128, 66, "any", 32), (129, 35, "any", 20), (100, 65, "any", 130)])
def test_many_clips_of_any_lengths(B, T, lens, D, dtype):
    """More clips than start at once, whatever order they are started in."""
    x = inputs(B, T, 2, 8, 16, D, dtype, seed=B)
    gen = torch.Generator().manual_seed(B)
    n = torch.full((B,), 17) if lens == "equal" else torch.randint(-3, T + 4, (B,), generator=gen)
    n = n.to(torch.int32)
    out = torch.full((B, T, 8, D), 5.0, dtype=dtype, device="cuda")
    got, end = operators.gated_delta(*x, lengths=n.cuda(), out=out)
    ref, rend = delta_rule(*x, lengths=n.clamp(0, T))
    on = (torch.arange(T)[None] < n[:, None]).cuda()
    assert bool((got[~on] == 5).all())
    near(torch.where(on[..., None, None], got, 0), ref, tol(T, 16), HALF_STEP[dtype], TINY[dtype])
    near(end, rend, tol(T, 16))
    alone = [operators.gated_delta(*(t[b:b + 1] for t in x), lengths=n[b:b + 1].cuda()) for b in (0, 1, B - 1)]
    for (o, e), b in zip(alone, (0, 1, B - 1)):
        assert torch.equal(e[0], end[b]) and torch.equal(o[0][on[b]], got[b][on[b]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("step", [0, 1, 5])
def test_one_frame_whose_step_says_nothing(step, dtype):
    """Tensors of one frame may have any stride from frame to frame."""
    x = inputs(2, 1, 1, 2, 24, 20, dtype, seed=step)
    ref, rend = delta_rule(*x)
    q, k, v = (t.as_strided(t.shape, (t.stride(0), step, *t.stride()[2:])) for t in x[:3])
    out = torch.full((2, 1, 2, 20), 7.0, dtype=dtype, device="cuda")
    got, end = operators.gated_delta(q, k, v, *x[3:], out=out.as_strided(out.shape, (40, step, 20, 1)))
    near(got, ref, tol(1, 24), HALF_STEP[dtype], TINY[dtype])
    near(end, rend, tol(1, 24))
    state = torch.zeros_like(end)
    got = operators.gated_delta_step(q, k, v, *x[3:], state, out=out.as_strided(out.shape, (40, step, 20, 1)))
    near(got, ref, tol(1, 24), HALF_STEP[dtype], TINY[dtype])
    near(state, rend, tol(1, 24))


@pytest.mark.gpu
def test_clips_without_a_frame():
    x = inputs(2, 4, 1, 1, 16, 16, F32)
    none = [t[:, :0] for t in x]
    state = torch.randn(2, 1, 16, 16, device="cuda")
    out, end = operators.gated_delta(*none, state=state)
    assert out.shape == (2, 0, 1, 16) and torch.equal(end, state)
    out, end = operators.gated_delta(*none)
    assert bool((end == 0).all())
    before = state.clone()
    assert operators.gated_delta_step(*none, state).shape == (2, 0, 1, 16) and torch.equal(state, before)
    out, end = operators.gated_delta(*[t[:0] for t in x])
    assert out.shape == (0, 4, 1, 16) and end.shape == (0, 1, 16, 16)


@pytest.mark.gpu
def test_streams_left_out_keep_their_rows():
    S, T, dtype = 6, 2, F16
    x = inputs(S, T, 2, 2, 32, 32, dtype, seed=5)
    on = torch.tensor([1, 0, 1, 1, 0, 0], dtype=torch.uint8)
    for t in x:
        t[on == 0] = math.nan
    state = torch.randn(S, 2, 32, 32, generator=torch.Generator().manual_seed(1)).cuda()
    state[1] = math.inf
    ref, rend = delta_rule(*[t[(on == 1).cuda()] for t in x], state=state[(on == 1).cuda()])
    for mask in (on, on.bool()):
        s, out = state.clone(), torch.full((S, T, 2, 32), 7.0, device="cuda", dtype=dtype)
        operators.gated_delta_step(*x, s, active=mask.cuda(), out=out)
        assert bool((out[(on == 0).cuda()] == 7.0).all()) and torch.equal(s[(on == 0).cuda()], state[(on == 0).cuda()])
        near(out[(on == 1).cuda()], ref, tol(T, 32), HALF_STEP[dtype], TINY[dtype])
        near(s[(on == 1).cuda()], rend, tol(T, 32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_any_strides(dtype):
    B, T, H, D = 2, 90, 2, 32
    q, k, v, g, beta = inputs(B, T, H, H, D, D, dtype, seed=6)
    ref, rend = operators.gated_delta(q, k, v, g, beta)
    fused = torch.cat((q, k, v), dim=-1)                                     # one projection's output, three views of it
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    frames_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    wide = torch.zeros(B, T, H, D + 3, device="cuda", dtype=dtype)           # rows at odd addresses
    odd = []
    for t in (q, k, v):
        w = wide.clone()
        w[..., 1:D + 1] = t
        odd.append(w[..., 1:D + 1])
    gates = [t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (g, beta)]
    for views in ([fused[..., :D], fused[..., D:2 * D], fused[..., 2 * D:]], heads_first, frames_first, odd):
        out = torch.zeros(B, H, T, 2 * D, device="cuda", dtype=dtype)
        got, end = operators.gated_delta(*views, *gates, out=out.transpose(1, 2)[..., :D])
        assert torch.equal(got, ref) and torch.equal(end, rend)
        assert bool((out[..., D:] == 0).all())
        s, s2 = torch.zeros_like(rend), torch.zeros_like(rend)
        a = operators.gated_delta_step(*[t[:, :3] for t in views], gates[0][:, :3], gates[1][:, :3], s)
        b = operators.gated_delta_step(q[:, :3], k[:, :3], v[:, :3], g[:, :3], beta[:, :3], s2)
        assert torch.equal(a, b) and torch.equal(s, s2)
    same = [t[:1].expand(B, -1, -1, -1) for t in (q, k, v)] + [t[:1].expand(B, -1, -1) for t in (g, beta)]
    out, end = operators.gated_delta(*same)                                  # one clip for every row of the batch: bit-identical rows
    assert torch.equal(out[0], out[1]) and torch.equal(end[0], end[1]) and torch.equal(out[0], ref[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cut", [1, 64, 100, 150])
def test_a_clip_in_two_calls_and_clip_against_steps(dtype, cut):
    x = inputs(2, 180, 2, 4, 64, 32, dtype, seed=8)
    ref, rend = delta_rule(*x)
    o1, s = operators.gated_delta(*[t[:, :cut] for t in x])
    o2, s2 = operators.gated_delta(*[t[:, cut:] for t in x], state=s, state_out=s)
    assert s2 is s
    near(torch.cat((o1, o2), 1), ref, tol(180, 64), HALF_STEP[dtype], TINY[dtype])
    near(s, rend, tol(180, 64))
    s = torch.zeros_like(s)
    o = torch.cat([operators.gated_delta_step(*[t[:, i:i + 60] for t in x], s) for i in range(0, 180, 60)], 1)
    near(o, ref, tol(180, 64), HALF_STEP[dtype], TINY[dtype])
    near(s, rend, tol(180, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("what, at", [("q", 70), ("k", 70), ("v", 70), ("g", 70), ("beta", 70), ("k", 0), ("v", 127), ("k", 129)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_non_finite_value_stays_where_it_belongs(dtype, what, at, value):
    x = inputs(2, 130, 2, 2, 32, 32, dtype, seed=11)
    clean, cend = operators.gated_delta(*x)
    y = [t.clone() for t in x]
    t = y["q k v g beta".split().index(what)]
    if what in ("g", "beta"):
        t[1, at, 0] = value
    else:
        t[1, at, 0, 5] = value
    out, end = operators.gated_delta(*y)
    hit = torch.zeros_like(out, dtype=torch.bool)
    if what == "q":
        hit[1, at, 0] = True
    elif what == "v":
        hit[1, at:, 0, 5] = True
    else:
        hit[1, at:, 0] = True
    assert torch.equal(out[~hit], clean[~hit])                # other clips, heads and earlier frames: bit for bit
    assert not bool(torch.isfinite(out[hit]).any())
    shit = torch.zeros_like(end, dtype=torch.bool)
    if what == "v":
        shit[1, 0, :, 5] = True
    elif what != "q":
        shit[1, 0] = True
    assert torch.equal(end[~shit], cend[~shit]) and not bool(torch.isfinite(end[shit]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_large_and_small_values_keep_their_precision(dtype):
    """Rows of v and states of very different size side by side: each column is as exact as it would be alone."""
    q, k, v, g, beta = inputs(1, 100, 1, 1, 64, 64, dtype, seed=12)
    size = 2.0 ** torch.linspace(-8, 8, 64).round().cuda()
    state = torch.randn(1, 1, 64, 64, generator=torch.Generator().manual_seed(1)).cuda() * size
    v = (v * size).to(dtype)
    out, end = operators.gated_delta(q, k, v, g, beta, state=state)
    ref, rend = delta_rule(q, k, v, g, beta, state=state)
    for c in range(64):
        near(out[..., c], ref[..., c], tol(100, 64), HALF_STEP[dtype], TINY[dtype])
        near(end[..., c], rend[..., c], tol(100, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_outputs_that_are_small_differences_of_large_terms(dtype):
    """A key that is written again takes back what it held: o = q S + P u, here (q = k, |k| = 1, beta = 1, no decay, scale 1: o = v) of terms `size` times
    the result.  An output takes Dk + 64 sums for these two and, through P (rows of norm sqrt(2) at most), Dk + 64 + 16 for u: 128 + 2 * 144 = 416
    roundings, each of at most half a step of fp32 of a partial sum, whose rms is `size`; signs are random, so the rms error is at
    most sqrt(416) u size, and the result's own rounding half a step / sqrt(3).  Terms of 16 bits would be off by 2^-16 of theirs, 4 to 5 times that."""
    B, T, H, D, size = 2, 64, 4, 64, 4096.0
    gen = torch.Generator().manual_seed(21)
    k = (torch.randint(0, 2, (B, T, H, D), generator=gen) * 2 - 1).to(dtype).cuda() / 8          # exact in every type, and so is its norm
    v = torch.randn(B, T, H, D, generator=gen).to(dtype).cuda()
    g, beta = torch.zeros(B, T, H, device="cuda"), torch.ones(B, T, H, device="cuda")
    state = size * torch.randn(B, H, D, D, generator=gen).cuda()
    ref, _ = delta_rule(k, k, v, g, beta, state=state, scale=1.0)
    assert float((ref - v.double().cpu()).abs().max()) < 1e-9
    out, _ = operators.gated_delta(k, k, v, g, beta, state=state, scale=1.0)
    off = float((out.double().cpu() - ref).square().mean().sqrt())
    own = HALF_STEP[dtype] / math.sqrt(3) * float(ref.square().mean().sqrt())
    bound = math.hypot(math.sqrt(416) * U * size, own)
    assert off <= bound, f"rms {off:.3g}, {off / bound:.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T, lens, Hk, Hv, Dk, Dv", [(1200, None, 1, 2, 64, 64), (2000, (2000, 777), 1, 1, 16, 40), (1500, (0, 1500), 2, 2, 128, 128), (900, (64, 899), 1, 2, 48, 20),
                                                     (1030, None, 1, 1, 100, 100)])
def test_few_long_clips_are_cut_into_segments(T, lens, Hk, Hv, Dk, Dv, dtype):
    """Against the definition, and against the same call without a workspace (one piece)."""
    B = 2
    x = inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=T, g_std=3.0)        # heads that remember a few frames beside heads that remember all
    x[3][0, T // 2] = -math.inf
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    state = 0.5 * torch.randn(B, Hv, Dk, Dv, generator=torch.Generator().manual_seed(1)).cuda()
    ref, rend = delta_rule(*x, state=state, lengths=lengths)
    out, end = operators.gated_delta(*x, state=state, lengths=lengths)
    near(out, ref, tol(T, Dk), HALF_STEP[dtype], TINY[dtype])
    near(end, rend, tol(T, Dk))
    q, k, v, g, beta = x
    L = backend.load_library()
    out1, end1 = torch.zeros_like(out), torch.empty_like(end)
    a = operators._GatedDeltaArgs({F32: 0, F16: 1, BF16: 2}[dtype], 0, B, T, Hk, Hv, Dk, Dv, 1 / math.sqrt(Dk), *[t.data_ptr() for t in x], out1.data_ptr(),
                                  q.stride()[:3], k.stride()[:3], v.stride()[:3], g.stride(), beta.stride(), out1.stride()[:3],
                                  state.data_ptr(), end1.data_ptr(), None if lens is None else lengths.data_ptr(), None)
    assert L.dpdf_gated_delta_workspace(0, ctypes.addressof(a)) > 0
    assert L.dpdf_gated_delta(0, ctypes.addressof(a), None, 0, torch.cuda.current_stream().cuda_stream) == 0
    near(out1, ref, tol(T, Dk), HALF_STEP[dtype], TINY[dtype])
    near(end1, rend, tol(T, Dk))


@pytest.mark.gpu
def test_captured_segments_update_a_state_in_place():
    """Replays go on from where the last one ended; the captured call's workspace is the graph's own."""
    x = inputs(2, 1200, 1, 2, 64, 64, BF16, seed=3, g_std=3.0)
    lengths = torch.tensor((1200, 100), dtype=torch.int32, device="cuda")
    state = torch.zeros(2, 2, 64, 64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        operators.gated_delta(*x, state=state.clone(), lengths=lengths)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:                                              # two of them, on the same state
        with torch.cuda.graph(g):
            outs.append(operators.gated_delta(*x, state=state, lengths=lengths, state_out=state)[0])
    mirror = 0.5 * torch.randn(2, 2, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    state.copy_(mirror)
    for r in range(4):
        x[2].copy_(torch.randn(2, 1200, 2, 64, generator=torch.Generator().manual_seed(r)))
        graphs[r % 2].replay()
        want, mirror = operators.gated_delta(*x, state=mirror, lengths=lengths)
        torch.cuda.synchronize()
        assert torch.equal(outs[r % 2], want) and torch.equal(state, mirror)


@pytest.mark.gpu
def test_a_workspace_over_the_lengths_is_refused():
    B, T, H, D = 1, 1200, 1, 64
    x = inputs(B, T, H, H, D, D, F32)
    out, end = torch.zeros(B, T, H, D, device="cuda"), torch.zeros(B, H, D, D, device="cuda")
    room = torch.zeros(1 << 20, dtype=torch.int32, device="cuda")
    strides = [(T * H * D, H * D, D)] * 3 + [(T * H, H, 1)] * 2 + [(T * H * D, H * D, D)]
    L = backend.load_library()
    for at in (0, 5):
        lengths = room[at:at + B]
        lengths.fill_(T)
        a = operators._GatedDeltaArgs(0, 0, B, T, H, H, D, D, 1.0, *[t.data_ptr() for t in x], out.data_ptr(), *strides, None, end.data_ptr(), lengths.data_ptr(), None)
        assert 0 < L.dpdf_gated_delta_workspace(0, ctypes.addressof(a)) <= 4 * room.numel()
        assert L.dpdf_gated_delta(0, ctypes.addressof(a), room.data_ptr(), 4 * room.numel(), torch.cuda.current_stream().cuda_stream) == -1
        assert "workspace overlaps" in L.dpdf_last_error().decode()
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((end == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B, T, lens, Hk, Hv, Dk, Dv", [(1, 1200, None, 1, 2, 64, 64), (3, 1500, (0, 200, 1500), 1, 2, 32, 40), (2, 1030, (1, 700), 2, 2, 128, 128),
                                                        (3, 900, (900, 0, 64), 1, 1, 100, 20)])
def test_segments_update_a_state_in_place(B, T, lens, Hk, Hv, Dk, Dv, dtype):
    """The first segment starts from the state that the last one, which has no frames in a short clip, writes over: the same bits as with two states."""
    x = inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=T, g_std=3.0)
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    state = 0.5 * torch.randn(B, Hv, Dk, Dv, generator=torch.Generator().manual_seed(1)).cuda()
    want, wend = operators.gated_delta(*x, state=state, lengths=lengths)
    near(wend, delta_rule(*x, state=state, lengths=lengths)[1], tol(T, Dk))
    for _ in range(5):
        s = state.clone()
        out, end = operators.gated_delta(*x, state=s, lengths=lengths, state_out=s)
        assert end is s and torch.equal(out, want) and torch.equal(s, wend)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Dv", [20, 60, 100])
@pytest.mark.parametrize("Dk", [20, 50, 100])
def test_long_clips_of_every_size(Dk, Dv, dtype):
    T = 600
    x = inputs(1, T, 1, 2, Dk, Dv, dtype, seed=Dk + Dv)
    state = 0.5 * torch.randn(1, 2, Dk, Dv, generator=torch.Generator().manual_seed(2)).cuda()
    out, end = operators.gated_delta(*x, state=state)
    ref, rend = delta_rule(*x, state=state)
    near(out, ref, tol(T, Dk), HALF_STEP[dtype], TINY[dtype])
    near(end, rend, tol(T, Dk))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["k", "v", "beta"])
@pytest.mark.parametrize("at", [0, 700, 1199])
def test_a_non_finite_value_in_a_clip_of_segments(what, at):
    x = inputs(1, 1200, 1, 2, 32, 32, BF16, seed=11)
    clean, cend = operators.gated_delta(*x)
    y = [t.clone() for t in x]
    if what == "beta":
        y[4][0, at, 0] = math.nan
    else:
        y["q k v".split().index(what)][0, at, 0, 5] = math.inf
    out, end = operators.gated_delta(*y)
    hit, shit = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(end, dtype=torch.bool)
    if what == "v":
        hit[0, at:, 0, 5] = shit[0, 0, :, 5] = True
    else:
        heads = slice(0, 2) if what == "k" else slice(0, 1)          # both value heads read the key head
        hit[0, at:, heads] = shit[0, heads] = True
    assert torch.equal(out[~hit], clean[~hit]) and not bool(torch.isfinite(out[hit]).any())
    assert torch.equal(end[~shit], cend[~shit]) and not bool(torch.isfinite(end[shit]).any())


@pytest.mark.gpu
def test_scale_is_the_callers():
    x = inputs(1, 70, 1, 1, 32, 32, F32)
    s = torch.zeros(1, 1, 32, 32, device="cuda")
    for scale in (0.0, 1.0, -2.5):
        ref, _ = delta_rule(*x, scale=scale)
        near(operators.gated_delta(*x, scale=scale)[0], ref, tol(70, 32))
        near(operators.gated_delta_step(*[t[:, :2] for t in x], s.clone(), scale=scale), ref[:, :2], tol(70, 32))


@pytest.mark.gpu
def test_refusals_of_device_tensors():
    q, k, v, g, beta = inputs(2, 8, 1, 2, 32, 32, BF16)
    state = torch.zeros(2, 2, 32, 32, device="cuda")
    bad = [dict(k=k[..., :16]), dict(k=k.float()), dict(v=v[:1]), dict(g=g.half()), dict(beta=beta.bfloat16()), dict(g=g[:, :, :1]), dict(state=state.half()),
           dict(state=state.transpose(2, 3)), dict(state=state[:1]), dict(lengths=torch.tensor([1, 2], device="cuda")), dict(lengths=torch.tensor([1, 2], dtype=torch.int32)),
           dict(out=torch.zeros(2, 8, 2, 32, device="cuda")), dict(out=v), dict(q=q.transpose(1, 3).contiguous().transpose(1, 3)), dict(scale=math.nan)]
    good = dict(q=q, k=k, v=v, g=g, beta=beta)
    for change in bad:
        with pytest.raises(ValueError):
            operators.gated_delta(**{**good, **change})
    with pytest.raises(ValueError, match="gradient"):
        operators.gated_delta(q, k, v.clone().requires_grad_(), g, beta)
    with torch.no_grad():
        operators.gated_delta(q, k, v.clone().requires_grad_(), g, beta)
    with pytest.raises(ValueError):
        operators.gated_delta_step(q, k, v, g, beta, state, active=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="head sizes"):
        operators.gated_delta(*inputs(1, 4, 1, 1, 144, 16, F32))
    both = torch.zeros(2 * 2 * 2 * 32 * 32, device="cuda")
    with pytest.raises(ValueError, match="in part"):
        operators.gated_delta(q, k, v, g, beta, state=both[:4096].view(2, 2, 32, 32), state_out=both[16:4112].view(2, 2, 32, 32))
    x, codes, scales = torch.zeros(2, 64, device="cuda"), torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), torch.zeros(4, 1, device="cuda")
    for change in (dict(codes=codes[:, :31]), dict(scales=scales.half()), dict(scales=scales[:, :0]), dict(zeros=scales), dict(bias=scales), dict(out=x), dict(codes=codes.int())):
        with pytest.raises(ValueError):
            operators.w4_matvec(**{**dict(x=x, codes=codes, scales=scales), **change})


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    """No derivative of either mode is computed, so that none is dropped silently."""
    from torch.autograd import forward_ad
    x = dict(zip("q k v g beta".split(), inputs(1, 3, 1, 2, 16, 16, F32)))
    state = torch.zeros(1, 2, 16, 16, device="cuda")
    y, codes, scales, _, bias = layer(2, 64, 8, 32, F32, False)
    out = torch.zeros(1, 3, 2, 16, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for n, t in x.items():
            with pytest.raises(ValueError, match="tangent"):
                operators.gated_delta(**{**x, n: dual(t)})
            with pytest.raises(ValueError, match="tangent"), torch.no_grad():
                operators.gated_delta_step(**{**x, n: dual(t)}, state=state)
        with pytest.raises(ValueError, match="tangent"):
            operators.gated_delta(**x, state=dual(state))
        with pytest.raises(ValueError, match="tangent"):
            operators.gated_delta(**x, out=dual(out))
        for change in (dict(x=dual(y)), dict(scales=dual(scales)), dict(bias=dual(bias))):
            with pytest.raises(ValueError, match="tangent"):
                operators.w4_matvec(**{**dict(x=y, codes=codes, scales=scales, bias=bias, group=32), **change})
        with pytest.raises(ValueError, match="tangent"):
            operators.w4_quantize(dual(y))
        operators.gated_delta(**x)                                # a level alone changes nothing
        operators.w4_matvec(y, codes, scales, group=32)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    far = 2 ** 31 + 64
    q, k, v, g, beta = inputs(2, 70, 1, 1, 32, 32, F16, seed=2)
    buf = torch.zeros(far + 70 * 96, dtype=F16, device="cuda")
    views = [buf.as_strided((2, 70, 1, 32), (far, 96, 32, 1), 32 * i) for i in range(3)]
    for a, b in zip(views, (q, k, v)):
        a.copy_(b)
    obuf = torch.zeros(far + 70 * 32, dtype=F16, device="cuda")
    ref, rend = operators.gated_delta(q, k, v, g, beta)
    out, end = operators.gated_delta(*views, g, beta, out=obuf.as_strided((2, 70, 1, 32), (far, 32, 32, 1)))
    assert torch.equal(out, ref) and torch.equal(end, rend)
    s = torch.zeros_like(end)
    s2 = s.clone()
    assert torch.equal(operators.gated_delta_step(*[t[:, :2] for t in views], g[:, :2], beta[:, :2], s),
                       operators.gated_delta_step(*[t[:, :2] for t in (q, k, v)], g[:, :2], beta[:, :2], s2)) and torch.equal(s, s2)
    del buf, obuf, views, out
    # a state of more than 2^31 values: the last stream's is right
    S = 4100
    x = inputs(1, 1, 1, 32, 128, 128, BF16, seed=3)
    wide = [t.expand(S, *t.shape[1:]) for t in x]
    state = torch.zeros(S, 32, 128, 128, device="cuda")
    state[0] = state[-1] = 0.25
    ref, rend = delta_rule(*x, state=state[-1:])
    out = operators.gated_delta_step(*wide, state)
    near(out[-1:], ref, tol(1, 128), HALF_STEP[BF16], TINY[BF16])
    near(state[-1:], rend, tol(1, 128))
    assert torch.equal(state[0], state[-1]) and torch.equal(out[0], out[-1])
    end = operators.gated_delta(*wide, state=state, state_out=state)[1]
    near(end[-1:], delta_rule(*x, state=rend.float())[1], 2 * tol(1, 128))


# ---------------------------------------------------------------------------------------------------------------------------------------
# GPU: 4-bit layers
# ---------------------------------------------------------------------------------------------------------------------------------------
def layer(M, K, N, group, dtype, zeros, seed=0, scale_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    groups = -(-K // group)
    x = torch.randn(M, K, generator=gen).to(dtype).cuda()
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=gen, dtype=torch.uint8).cuda()
    scales = (0.01 + torch.rand(N, groups, generator=gen)).to(scale_dtype or dtype).cuda()
    z = torch.randint(0, 16, (N, groups), generator=gen, dtype=torch.uint8).cuda() if zeros else None
    return x, codes, scales, z, torch.randn(N, generator=gen).to(dtype).cuda()


def near_layer(y, ref, mag, K, dtype):
    """A sum of K products and its pieces: 8 deviations of sqrt(K + 16) roundings of the magnitudes' sum, which bounds every partial sum; codes
    with a zero of up to 15 may be taken apart into code and zero, which doubles the magnitudes at most threefold."""
    bound = 8 * math.sqrt(K + 16) * U * 4 * mag + HALF_STEP[dtype] * ref.abs() * 1.01 + TINY[dtype]
    off = (y.double().cpu() - ref).abs()
    assert bool((off <= bound).all()), f"worst {float((off / bound).max()):.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M, K, N, group", [(1, 1, 1, 32), (1, 2, 3, 32), (2, 31, 17, 32), (1, 64, 64, 64), (3, 100, 50, 32), (1, 256, 768, 64), (4, 255, 33, 128), (7, 513, 100, 64),
                                            (8, 1024, 96, 128), (9, 300, 31, 96), (16, 2048, 130, 32), (17, 640, 64, 640), (33, 333, 77, 64), (1, 8192, 48, 128), (5, 4096, 16, 4096),
                                            (2, 160, 64, 1024)])
def test_w4_layers_against_the_definition(M, K, N, group, dtype):
    for zeros in (False, True):
        x, codes, scales, z, bias = layer(M, K, N, group, dtype, zeros, seed=K + M)
        for b in (None, bias):
            ref, mag = w4_layer(x, codes, scales, z, b, group)
            near_layer(operators.w4_matvec(x, codes, scales, zeros=z, bias=b, group=group), ref, mag, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, scale_dtype", [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("M, N", [(3, 1000), (2, 16400), (17, 8200), (5, 32800), (40, 11000)])
@pytest.mark.parametrize("K, group", [(130, 32), (700, 64), (1300, 128), (1100, 96)])
def test_w4_layers_of_many_outputs(M, N, K, group, dtype, scale_dtype):
    """Every number of tiles to a workgroup, of waves and of blocks to a wave; rows of x in more than one tile."""
    x, codes, scales, z, bias = layer(M, K, N, group, dtype, K == 700, seed=N, scale_dtype=scale_dtype)
    y = operators.w4_matvec(x, codes, scales, zeros=z, bias=bias, group=group)
    at = torch.cat([torch.arange(0, N, 97), torch.arange(N - 40, N)]).cuda()             # outputs are independent: some of all tiles, and the last
    ref, mag = w4_layer(x, codes[at], scales[at], None if z is None else z[at], bias[at], group)
    near_layer(y[:, at], ref, mag, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_w4_strides_alignments_and_scale_types(dtype):
    M, K, N, group = 5, 384, 70, 64
    x, codes, scales, z, bias = layer(M, K, N, group, dtype, True, scale_dtype=F32)
    ref, mag = w4_layer(x, codes, scales, z, bias, group)
    near_layer(operators.w4_matvec(x, codes, scales, zeros=z, bias=bias, group=group), ref, mag, K, dtype)
    near_layer(operators.w4_matvec(x[0], codes, scales, zeros=z, bias=bias, group=group), ref[0], mag[0], K, dtype)
    near_layer(operators.w4_matvec(x[:1].expand(M, -1), codes, scales, zeros=z, bias=bias, group=group), ref[:1].expand(M, -1), mag[:1].expand(M, -1), K, dtype)
    for off, pitch in ((0, 208), (1, 200), (4, 196), (8, 200), (16, 224)):
        buf = torch.zeros(N * pitch + 32, dtype=torch.uint8, device="cuda")
        c = buf.as_strided((N, K // 2), (pitch, 1), off)
        c.copy_(codes)
        xw = torch.zeros(M, K + 11, dtype=dtype, device="cuda")
        xw[:, off % 8:off % 8 + K] = x
        xw[:, off % 8 + K:] = math.nan                        # behind a row: never read
        sw = torch.full((N, K // group + off), math.nan, device="cuda")
        sw[:, off:] = scales
        zw = torch.full((N, K // group + off), 99, dtype=torch.uint8, device="cuda")
        zw[:, off:] = z
        out = torch.full((M, N + 5), 7.0, dtype=dtype, device="cuda")
        operators.w4_matvec(xw[:, off % 8:off % 8 + K], c, sw[:, off:], zeros=zw[:, off:], bias=bias, group=group, out=out[:, 2:N + 2])
        near_layer(out[:, 2:N + 2], ref, mag, K, dtype)
        assert bool((out[:, :2] == 7).all()) and bool((out[:, N + 2:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 6, 20])
def test_w4_rows_are_independent_and_repeat(dtype, M):
    x, codes, scales, z, _ = layer(M, 1000, 90, 128, dtype, True)
    y = operators.w4_matvec(x, codes, scales, zeros=z, group=128)
    assert torch.equal(y, operators.w4_matvec(x, codes, scales, zeros=z, group=128))
    bad = x.clone()
    bad[M - 1, 7], bad[M - 1, 900] = math.nan, math.inf
    got = operators.w4_matvec(bad, codes, scales, zeros=z, group=128)
    assert torch.equal(got[:M - 1], y[:M - 1]) and not bool(torch.isfinite(got[M - 1]).any())
    s = scales.clone()
    s[5, 2] = math.inf                                        # one output's weights
    got = operators.w4_matvec(x, codes, s, zeros=z, group=128)
    keep = torch.arange(90) != 5
    assert torch.equal(got[:, keep], y[:, keep]) and not bool(torch.isfinite(got[:, 5]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scales32", [True, False])
@pytest.mark.parametrize("M, K, N, group", [(3, 1300, 5000, 32), (3, 1300, 5000, 64), (3, 1300, 5000, 128), (20, 700, 4000, 96), (2, 4100, 20000, 128), (9, 4096, 20480, 128),
                                            (9, 4100, 14000, 128), (9, 1300, 14000, 64), (1, 300, 70000, 32)])
def test_w4_layers_between_the_splits(M, K, N, group, scales32, dtype):
    """One, two and four tiles to a workgroup and four and eight waves, by tiles for each CU: 1.2, 1.9, 2 - 5, 17."""
    x, codes, scales, z, bias = layer(M, K, N, group, dtype, group == 64, seed=N, scale_dtype=F32 if scales32 else None)
    y = operators.w4_matvec(x, codes, scales, zeros=z, bias=bias, group=group)
    at = torch.cat([torch.arange(0, N, 997), torch.arange(N - 40, N)]).cuda()
    ref, mag = w4_layer(x, codes[at], scales[at], None if z is None else z[at], bias[at], group)
    near_layer(y[:, at], ref, mag, K, dtype)
    assert torch.equal(y, operators.w4_matvec(x, codes, scales, zeros=z, bias=bias, group=group))


def near_sparse_layer(y, x, codes, scales, z, group, dtype):
    """Weights near their zero: a term whose code is the zero is 0 and adds nothing, the n others of an output are at most three products each (fp32 rows
    are three limbs) with one sum each, and a scale and a sum per group: 8 deviations of sqrt(5 n) roundings of the terms' magnitudes."""
    ref, mag = w4_layer(x, codes, scales, z, None, group)
    k = torch.arange(x.shape[-1])
    code = (codes.cpu()[:, k // 2].int() >> (4 * (k % 2))) & 15
    n = (code != (8 if z is None else z.cpu()[:, k // group].int())).sum(1).double()
    bound = 8 * (5 * n).sqrt() * U * mag + HALF_STEP[dtype] * ref.abs() * 1.01 + TINY[dtype] * (n > 0)
    off = (y.double().cpu() - ref).abs()
    assert bool((off <= bound).all()), f"worst {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M, K, N, group", [(1, 4096, 48, 64), (5, 1000, 40, 32), (16, 2048, 40, 128), (3, 301, 20, 96)])
@pytest.mark.parametrize("zero", [None, 0, 3, 11, 15])
def test_w4_weights_near_their_zero(M, K, N, group, zero, dtype):
    """Rows of nothing but zeros (0, exactly), of one weight, of a few, of weights close around the zero."""
    gen = torch.Generator().manual_seed(K + (zero or 0))
    x, _, scales, _, bias = layer(M, K, N, group, dtype, False, seed=K)
    at = 8 if zero is None else zero
    code = torch.full((N, K + K % 2), at)
    for n in range(N):
        if n % 4 == 1:
            code[n, torch.randint(0, K, (1,), generator=gen)] = (at + 1 + n) % 16
        elif n % 4 == 2:
            code[n, torch.randint(0, K, (7,), generator=gen)] = torch.randint(0, 16, (7,), generator=gen)
        elif n % 4 == 3:
            code[n] = (at + (0.7 * torch.randn(K + K % 2, generator=gen)).round().long()).clamp(0, 15)
    codes = (code[:, ::2] | code[:, 1::2] << 4).to(torch.uint8).cuda()
    z = None if zero is None else torch.full(scales.shape, zero, dtype=torch.uint8, device="cuda")
    y = operators.w4_matvec(x, codes, scales, zeros=z, group=group)
    near_sparse_layer(y, x, codes, scales, z, group, dtype)
    assert bool((y[:, ::4] == 0).all())
    yb = operators.w4_matvec(x, codes, scales, zeros=z, bias=bias, group=group)
    assert torch.equal(yb[:, ::4], bias[::4].expand(M, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_zeros_above_15_show(group, dtype):
    x, codes, scales, z, _ = layer(2, 610, 60, group, dtype, True, seed=group)
    y = operators.w4_matvec(x, codes, scales, zeros=z, group=group)
    hit = torch.zeros(60, dtype=torch.bool, device="cuda")
    for n, at, v in ((3, 0, 16), (20, 1, 255), (40, scales.shape[1] - 1, 128), (59, 2, 31)):
        z[n, at] = v
        hit[n] = True
    got = operators.w4_matvec(x, codes, scales, zeros=z, group=group)
    assert torch.equal(got[:, ~hit], y[:, ~hit]) and bool(got[:, hit].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_w4_large_inputs_are_not_taken_out_of_range(dtype):
    """|x| of 2e37, two in a row: their products with code - zero, 8 at most, stay below 3.4e38, and so does their sum."""
    x, codes, scales, _, _ = layer(4, 640, 40, 64, dtype, False, seed=5)
    keep = torch.zeros_like(x)
    keep[:, [3, 630]] = torch.tensor([1.0, -1.0], device="cuda", dtype=dtype)
    x = keep * 2e37
    near_sparse_layer(operators.w4_matvec(x, codes, scales), x, codes, scales, None, 64, dtype)


@pytest.mark.gpu
def test_w4_empty_batch_and_far_offsets():
    x, codes, scales, z, bias = layer(3, 128, 40, 64, F16, False)
    assert operators.w4_matvec(x[:0], codes, scales).shape == (0, 40)
    buf = torch.zeros(2 * (2 ** 31 + 16) + 64, dtype=torch.uint8, device="cuda")        # rows of codes 2 GiB apart
    c = buf.as_strided((3, 64), (2 ** 31 + 16, 1))
    c.copy_(codes[:3])
    assert torch.equal(operators.w4_matvec(x, c, scales[:3]), operators.w4_matvec(x, codes[:3].contiguous(), scales[:3]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("N, K, group", [(5, 64, 64), (33, 257, 32), (16, 1000, 128), (3, 1, 32), (64, 512, 4096)])
def test_w4_quantize_is_the_formula(dtype, N, K, group):
    gen = torch.Generator().manual_seed(K)
    w = torch.randn(N, K, generator=gen).to(dtype)
    w[0] = 0                                                  # a group of nothing
    w[-1] = w[-1].abs()                                       # a group of one sign
    if K > 60:
        w[1, :14] = torch.arange(14).to(dtype) / 2 - 3.25     # ties
    groups = -(-K // group)
    pad = torch.nn.functional.pad(w.float(), [0, groups * group - K]).view(N, groups, group)
    for symmetric in (False, True):
        codes, scales, zeros = operators.w4_quantize(w.cuda(), group=group, symmetric=symmetric)
        lo, hi = pad.amin(-1).clamp_max(0), pad.amax(-1).clamp_min(0)
        s = (torch.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15).to(dtype)
        f = s.float()
        z = torch.full_like(f, 8.0) if symmetric else torch.where(f > 0, (-lo / f).round().clamp(0, 15), 0.0)
        c = torch.where(f[..., None] > 0, (pad / f[..., None]).round() + z[..., None], z[..., None]).clamp(0, 15).view(N, -1)[:, :K].to(torch.uint8)
        assert scales.dtype == dtype and torch.equal(scales.cpu(), s)
        assert (zeros is None) == symmetric and (symmetric or torch.equal(zeros.cpu().float(), z))
        got = torch.stack((codes.cpu() & 15, codes.cpu() >> 4), -1).flatten(1)
        assert codes.shape == (N, (K + 1) // 2) and codes.stride(0) % 16 == 0 and torch.equal(got[:, :K], c)
        y, mag = w4_layer(torch.eye(K), codes, scales, zeros, None, group)
        step = f.double().repeat_interleave(group, 1)[:, :K].t()
        assert bool(((y - w.double().t()).abs() <= step * 0.5 * 1.1 + step * 8 * HALF_STEP[dtype] * 2).all())        # half a step, and the scale's own rounding over 8 to 15 steps


@pytest.mark.gpu
def test_w4_quantize_of_more_groups_than_a_launch_has_waves():
    N, K = 2 ** 21 + 5, 1024
    w = torch.empty(N, K, dtype=BF16, device="cuda")
    w[:-9] = torch.randn(1, K, generator=torch.Generator().manual_seed(1)).cuda()
    w[-9:] = torch.randn(9, K, generator=torch.Generator().manual_seed(2)).cuda()
    codes, scales, zeros = operators.w4_quantize(w, group=32)
    for rows in (slice(0, 3), slice(2 ** 20, 2 ** 20 + 3), slice(N - 9, N)):
        c, s, z = operators.w4_quantize(w[rows].clone(), group=32)
        assert torch.equal(codes[rows], c) and torch.equal(scales[rows], s) and torch.equal(zeros[rows], z)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_w4_quantize_shows_weights_that_are_not_finite(value, symmetric, dtype):
    """The group's scale is NaN, its codes are the zero, every other group is what it was; the layer's outputs of that row are NaN."""
    w = torch.randn(6, 200, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    codes, scales, zeros = operators.w4_quantize(w, symmetric=symmetric)
    hit = torch.zeros_like(scales, dtype=torch.bool)
    for n, k in ((1, 0), (2, 63), (3, 130), (5, 199)):
        w[n, k] = value
        hit[n, k // 64] = True
    got, gs, gz = operators.w4_quantize(w, symmetric=symmetric)
    assert bool(gs[hit].isnan().all()) and torch.equal(gs[~hit], scales[~hit])
    cols = hit.repeat_interleave(32, 1)[:, :100]
    assert torch.equal(got[~cols], codes[~cols]) and bool((got[cols] == (0x88 if symmetric else 0)).all())
    if not symmetric:
        assert torch.equal(gz[~hit], zeros[~hit]) and bool((gz[hit] == 0).all())
    y = operators.w4_matvec(torch.ones(2, 200, dtype=dtype, device="cuda"), got, gs, zeros=gz)
    assert torch.equal(y.isnan(), hit.any(1).expand(2, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_w4_quantize_of_a_range_that_fp32_does_not_hold(dtype):
    """A group from -3e38 to 3e38: finite weights, a finite scale.  Its step is 4e37, half of it the most that a weight is off (and the scale's rounding over 8 steps)."""
    w = torch.linspace(-3e38, 3e38, 64, dtype=torch.float64).to(dtype)[None]        # in fp32 linspace itself overflows
    codes, scales, zeros = operators.w4_quantize(w.cuda())
    assert bool(scales.isfinite().all())
    y, _ = w4_layer(torch.eye(64), codes, scales, zeros, None, 64)
    step = float(scales.double())
    assert abs(step / 4e37 - 1) < 0.01
    assert float((y.t() - w.double()).abs().max()) <= step * (0.5 * 1.1 + 16 * HALF_STEP[dtype])


# ---------------------------------------------------------------------------------------------------------------------------------------
# GPU: together, on streams, in graphs
# ---------------------------------------------------------------------------------------------------------------------------------------
class Layer:
    """A recurrent layer of a live stream as a program would build it: 4-bit projections of a frame to q, k, v and the gates, the recurrence, and a
    4-bit projection back."""

    def __init__(self, dtype, width=128, heads=2, dim=32, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.dim, n = heads, dim, heads * dim
        self.inw = (torch.randn(3 * n + 2 * heads, width, generator=gen) / math.sqrt(width)).to(dtype).cuda()
        self.outw = (torch.randn(width, n, generator=gen) / math.sqrt(n)).to(dtype).cuda()
        self.inq, self.outq = operators.w4_quantize(self.inw, group=32), operators.w4_quantize(self.outw, group=32)

    def parts(self, y):
        """[S, T, 3 n + 2 heads] -> q, k, v, g, beta"""
        n = self.heads * self.dim
        q, k, v = (y[..., i * n:(i + 1) * n].unflatten(-1, (self.heads, self.dim)) for i in range(3))
        unit = [torch.nn.functional.normalize(t.float(), dim=-1).to(y.dtype) for t in (q, k)]
        g, b = y[..., 3 * n:].float().chunk(2, -1)
        return (*unit, v, -torch.nn.functional.softplus(g), torch.sigmoid(b))

    def project(self, x, w):
        return operators.w4_matvec(x.reshape(-1, x.shape[-1]), w[0], w[1], zeros=w[2], group=32).view(*x.shape[:-1], -1)

    def clip(self, x):
        o, s = operators.gated_delta(*self.parts(self.project(x, self.inq)))
        return self.project(o.flatten(2), self.outq), s

    def hop(self, x, state):
        o = operators.gated_delta_step(*self.parts(self.project(x, self.inq)), state)
        return self.project(o.flatten(2), self.outq)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_layer_over_clips_is_the_layer_hop_by_hop(dtype):
    lay = Layer(dtype)
    x = torch.randn(3, 70, 128, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    y, end = lay.clip(x)
    state = torch.zeros_like(end)
    hops = torch.cat([lay.hop(x[:, t:t + 1], state) for t in range(70)], 1)
    # projections of one frame and of all are the same sums in one order or another; the recurrence's outputs are rounded to the type between
    # the two projections, where one step's difference reaches the sums of 64 products
    step = 2 * HALF_STEP[dtype]
    near(hops, y.double().cpu(), 2 * tol(70, 32) + step, step)
    near(state, end.double().cpu(), 2 * tol(70, 32) + (step if dtype != F32 else 0))
    # and the whole against 64 bits, from the values that the codes stand for
    (ci, si, zi), (co, so, zo) = lay.inq, lay.outq
    p = w4_layer(x.flatten(0, 1), ci, si, zi, None, 32)[0].view(3, 70, -1).to(dtype).cuda()
    o, rend = delta_rule(*lay.parts(p))
    r = w4_layer(o.to(dtype).flatten(0, 1).flatten(1), co, so, zo, None, 32)[0].view(3, 70, -1)
    near(y, r, 2 * tol(70, 32) + step, step)


@pytest.mark.gpu
def test_calls_on_other_streams_and_two_at_once():
    lay = Layer(BF16)
    xs = [torch.randn(2, 200, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    want = [lay.clip(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(lay.clip(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y, e in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(e, want[i][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_calls_replay(dtype):
    S = 5
    lay = Layer(dtype)
    x = torch.randn(S, 1, 128, device="cuda").to(dtype)
    clip = torch.randn(2, 300, 128, device="cuda").to(dtype)
    state = torch.zeros(S, 2, 32, 32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lay.hop(x, state.clone()); lay.clip(clip)
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y = lay.hop(x, state)
    with torch.cuda.graph(g2):
        yc, ec = lay.clip(clip)
    mirror = torch.zeros_like(state)
    state.zero_()
    for r in range(4):
        x.copy_(torch.randn(S, 1, 128, generator=torch.Generator().manual_seed(r)))
        clip.copy_(torch.randn(2, 300, 128, generator=torch.Generator().manual_seed(50 + r)))
        g1.replay(); g2.replay()
        want, (wc, we) = lay.hop(x, mirror), lay.clip(clip)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, mirror) and torch.equal(yc, wc) and torch.equal(ec, we)
