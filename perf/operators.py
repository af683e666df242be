"""Cases of the stand-alone operators (`dpdfnet_amd.operators`): the gated delta rule over whole clips and hop by hop, and dense layers
with 4-bit weights for a few rows.  `run` computes a case with elementary torch operations, or, where `own` is true, with the calls that a
program makes of the operators."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64        # frames of a chunk in the plain form of the gated delta rule


# ---------------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------------
def _clip(name, B, T, Hk, Hv, Dk, Dv, dtype, ragged=False, state=False):
    return {"name": name, "op": "clip", "B": B, "T": T, "Hk": Hk, "Hv": Hv, "Dk": Dk, "Dv": Dv, "dtype": dtype, "ragged": ragged, "state": state}


def _hop(name, S, T, Hk, Hv, Dk, Dv, dtype, masked=False):
    return {"name": name, "op": "hop", "S": S, "T": T, "Hk": Hk, "Hv": Hv, "Dk": Dk, "Dv": Dv, "dtype": dtype, "masked": masked}


def _w4(name, M, K, N, group, dtype, zeros=False, bias=False):
    return {"name": name, "op": "w4", "M": M, "K": K, "N": N, "group": group, "dtype": dtype, "zeros": zeros, "bias": bias}


def listed():
    return [
        # 256 clips of 10 s (1003 frames), 256 channels as four heads of 64: the batch that a directory of files makes, clips of many lengths
        _clip("clips_256x1003_bf16", 256, 1003, 4, 4, 64, 64, "bf16", ragged=True),
        # 16 clips of 10 s in full precision, going on from a state; two value heads share a key head
        _clip("clips_16x1003_fp32", 16, 1003, 2, 4, 64, 64, "fp32", state=True),
        # one recording of 164 s, wide heads: few sequences, a long dependent chain
        _clip("recording_1x16384_bf16", 1, 16384, 8, 16, 128, 128, "bf16"),
        # clips shorter than a second, odd head sizes
        _clip("short_3x77_fp16", 3, 77, 2, 6, 48, 80, "fp16", ragged=True, state=True),
        # one live stream, one hop: latency
        _hop("hop_1_fp32", 1, 1, 4, 4, 64, 64, "fp32"),
        # a pool of 512 streams of which most have a hop
        _hop("hop_512_bf16", 512, 1, 4, 4, 64, 64, "bf16", masked=True),
        # 192 streams with wide heads, two hops at once: the state's bytes are all that counts
        _hop("hop_192x2_bf16", 192, 2, 16, 32, 128, 128, "bf16"),
        # the gate matrix of a GRU of 256 for one stream: latency
        _w4("w4_1x256x768_fp32", 1, 256, 768, 64, "fp32", bias=True),
        # one stream through a layer of some size
        _w4("w4_1x4096x16384_bf16", 1, 4096, 16384, 128, "bf16"),
        # odd sizes: a last group that is not whole, rows that end inside a byte's pair
        _w4("w4_5x1003x777_fp16", 5, 1003, 777, 32, "fp16", zeros=True, bias=True),
        # 16 streams
        _w4("w4_16x4096x4096_fp16", 16, 4096, 4096, 64, "fp16", zeros=True),
        # eight streams through a large layer
        _w4("w4_8x8192x32768_bf16", 8, 8192, 32768, 128, "bf16", zeros=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    op = rng.choice(["clip", "hop", "w4"])
    if op == "w4":
        M, K = _log_int(rng, 1, 32), _log_int(rng, 100, 8192)
        N = _log_int(rng, 100, 32768)
        if rng.random() < 0.5:            # a layer's usual sizes are multiples of 64, the other half is odd
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        c = _w4("", M, K, N, rng.choice([32, 64, 128]), dtype, rng.random() < 0.5, rng.random() < 0.5)
    else:
        Dk = rng.choice([16, 24, 32, 48, 64, 64, 64, 80, 96, 128, 128])
        Dv = Dk if rng.random() < 0.6 else rng.choice([16, 32, 40, 64, 100, 128])
        Hk, share = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3])
        Hv = Hk * share
        if op == "hop":
            S = max(1, min(_log_int(rng, 1, 1024), 192 * 32 * 128 * 128 // (Hv * Dk * Dv)))
            c = _hop("", S, rng.choice([1, 1, 1, 2, 3, 4]), Hk, Hv, Dk, Dv, dtype, rng.random() < 0.4)
        else:
            T = _log_int(rng, 30, 4096)
            B = max(1, min(_log_int(rng, 1, 256), 128 * 1003 * 4 * 64 // (T * Hv * max(Dk, Dv))))
            c = _clip("", B, T, Hk, Hv, Dk, Dv, dtype, rng.random() < 0.5, rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(c):
    """The clips' lengths: from the whole of T down to about a third of it, and one clip without a frame where there are three or more."""
    B, T = c["B"], c["T"]
    if not c["ragged"]:
        return [T] * B
    return [T if b == 0 else 0 if b == 2 else max(1, T - (b * 197) % max(1, 2 * T // 3)) for b in range(B)]


def _active(c):
    return [not (c["masked"] and s % 5 == 3) for s in range(c["S"])]


# ---------------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "w4":
        M, K, N, group = case["M"], case["K"], case["N"], case["group"]
        groups = -(-K // group)
        st = {"case": case, "x": randn(M, K).to(dt),
              "codes": torch.randint(0, 256, (N, -(-K // 2)), device="cuda", dtype=torch.uint8, generator=gen),
              "scales": ((0.5 + torch.rand(N, groups, device="cuda", generator=gen)) * (0.3 / math.sqrt(K))).to(dt),
              "zeros": None, "bias": randn(N).to(dt) if case["bias"] else None}
        if case["zeros"]:
            st["zeros"] = torch.randint(4, 12, (N, groups), device="cuda", dtype=torch.uint8, generator=gen)
        return st
    T, Hk, Hv, Dk, Dv = (case[n] for n in ("T", "Hk", "Hv", "Dk", "Dv"))
    B = case["B"] if case["op"] == "clip" else case["S"]
    unit = torch.nn.functional.normalize
    st = {"case": case,
          "q": unit(randn(B, T, Hk, Dk), dim=-1).to(dt), "k": unit(randn(B, T, Hk, Dk), dim=-1).to(dt), "v": randn(B, T, Hv, Dv).to(dt),
          # a head's memory lasts from a few frames to some thousand
          "g": -torch.exp(2.0 * randn(1, 1, Hv) - 4.0) * torch.rand(B, T, Hv, device="cuda", generator=gen),
          "beta": torch.sigmoid(randn(B, T, Hv))}
    if case["op"] == "hop":
        st["state"] = 0.3 * randn(B, Hv, Dk, Dv)
        st["active"] = torch.tensor(_active(case), device="cuda", dtype=torch.uint8) if case["masked"] else None
    else:
        st["state"] = 0.3 * randn(B, Hv, Dk, Dv) if case["state"] else None
        st["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
    # what a call leaves unwritten (frames behind a clip's end, streams without a hop) keeps these zeros
    st["out"] = torch.zeros(B, T, Hv, Dv, device="cuda", dtype=dt)
    return st


# ---------------------------------------------------------------------------------------------------------------------------------------
# the operators' calls and their plain forms
# ---------------------------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from dpdfnet_amd import operators
        if op == "w4":
            return operators.w4_matvec(s["x"], s["codes"], s["scales"], zeros=s["zeros"], bias=s["bias"], group=s["case"]["group"])
        if op == "hop":
            return operators.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], active=s["active"], out=s["out"]), s["state"]
        return operators.gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], state=s["state"], lengths=s["lengths"], out=s["out"])
    return {"w4": _plain_w4, "hop": _plain_hop, "clip": _plain_clip}[op](s)


def _plain_w4(s):
    x, codes, group = s["x"], s["codes"], s["case"]["group"]
    K = x.shape[1]
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1)[:, :K].float()
    at = torch.arange(K, device=x.device) // group
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, at]
    y = x.float() @ ((q - zero) * s["scales"].float()[:, at]).t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(x.dtype)


def _plain_hop(s):
    share = s["case"]["Hv"] // s["case"]["Hk"]
    q, k = (s[n].float().repeat_interleave(share, dim=2) for n in ("q", "k"))
    v, state, outs = s["v"].float(), s["state"], []
    S = state
    for t in range(v.shape[1]):            # a recurrence: every hop needs the one before
        S = S * s["g"][:, t].exp()[..., None, None]
        e = s["beta"][:, t, :, None] * (v[:, t] - (S * k[:, t, :, :, None]).sum(2))
        S = S + k[:, t, :, :, None] * e[:, :, None]
        outs.append((S * q[:, t, :, :, None]).sum(2) / math.sqrt(q.shape[-1]))
    o = torch.stack(outs, dim=1).to(s["out"].dtype)
    if s["active"] is None:
        state.copy_(S)
        s["out"].copy_(o)
    else:
        on = s["active"].bool()[:, None, None, None]
        state.copy_(torch.where(on, S, state))
        s["out"].copy_(torch.where(on, o, s["out"]))
    return s["out"], state


def _plain_clip(s):
    """The recurrence in chunks of 64 frames: inside a chunk the frames' corrections are the solution u of a unit lower triangular system,
    (I + A) u = beta (v - decay k S), and the chunks follow each other through the state S."""
    c = s["case"]
    B, T, Hv, Dk, Dv, share = c["B"], c["T"], c["Hv"], c["Dk"], c["Dv"], c["Hv"] // c["Hk"]
    n = -(-T // CHUNK)
    lengths = s["lengths"]
    live = None if lengths is None else (torch.arange(T, device="cuda")[None] < lengths[:, None])

    def chunks(x, share=1):                # [B, T, H, ..] -> [n, B, Hv, CHUNK, ..], nothing behind a clip's end
        if live is not None:
            x = x * live.view(B, T, *([1] * (x.dim() - 2)))
        x = torch.nn.functional.pad(x, [0, 0] * (x.dim() - 2) + [0, n * CHUNK - T])
        x = x.unflatten(1, (n, CHUNK)).repeat_interleave(share, dim=3)
        return x.movedim(1, 0).transpose(2, 3).contiguous()

    q, k, v = chunks(s["q"].float(), share), chunks(s["k"].float(), share), chunks(s["v"].float())
    gam = chunks(s["g"].double()).cumsum(-1)            # 64 bits: what counts is the small difference of two long sums
    beta = chunks(s["beta"])[..., None]
    lower = torch.ones(CHUNK, CHUNK, device="cuda", dtype=torch.bool).tril()
    decay = torch.where(lower, gam[..., :, None] - gam[..., None, :], -math.inf).exp().float()
    kt = k.transpose(-1, -2).contiguous()
    A = beta * decay.tril(-1) * (k @ kt)
    P = decay * (q @ kt) / math.sqrt(Dk)
    G, end = gam.exp().float()[..., None], (gam[..., -1:] - gam).exp().float()[..., None]
    inv = torch.eye(CHUNK, device="cuda").expand_as(A)
    at = torch.arange(CHUNK, device="cuda")
    size = 1
    while size < CHUNK:                    # the inverse of I + A from those of its diagonal blocks, twice the size each time
        below = (at[:, None] // size % 2 == 1) & (at[:, None] // size - 1 == at[None] // size)
        inv = inv - inv @ (A * below) @ inv
        size *= 2
    S = torch.zeros(B, Hv, Dk, Dv, device="cuda") if s["state"] is None else s["state"]
    outs = []
    for i in range(n):                     # a recurrence: every chunk needs the one before
        u = inv[i] @ (beta[i] * (v[i] - G[i] * (k[i] @ S)))
        outs.append(G[i] * (q[i] @ S) / math.sqrt(Dk) + P[i] @ u)
        S = G[i][..., -1:, :] * S + kt[i] @ (end[i] * u)
    o = torch.stack(outs, dim=1).transpose(2, 3).reshape(B, n * CHUNK, Hv, Dv)[:, :T].to(s["out"].dtype)
    s["out"].copy_(o if live is None else torch.where(live[..., None, None], o, s["out"]))
    return s["out"], S


# ---------------------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "w4":
        M, K, N = case["M"], case["K"], case["N"]
        groups = -(-K // case["group"])
        b = N * -(-K // 2) + N * groups * (e + (1 if case["zeros"] else 0)) + M * (K + N) * e + (N * e if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * M * K * N}
    Hk, Hv, Dk, Dv = (case[n] for n in ("Hk", "Hv", "Dk", "Dv"))
    if case["op"] == "hop":
        seqs = sum(_active(case))
        frames, states = seqs * case["T"], 2 * seqs
    else:
        seqs = case["B"]
        frames, states = sum(_lengths(case)), seqs * (2 if case["state"] else 1)
    b = frames * (2 * Hk * Dk * e + 2 * Hv * Dv * e + 2 * Hv * 4) + states * Hv * Dk * Dv * 4
    return {"bytes": b, "flops": frames * Hv * 6 * Dk * Dv}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "w4":
        K = case["K"]
        k = torch.arange(K, device="cuda")
        code = (s["codes"][:, k // 2].to(torch.int32) >> (4 * (k % 2))) & 15
        zero = 8 if s["zeros"] is None else s["zeros"].to(torch.int32)[:, k // case["group"]]
        y = s["x"].double() @ ((code - zero).double() * s["scales"].double()[:, k // case["group"]]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    B, T, Hv, Dv = s["v"].shape
    Dk = case["Dk"]
    head = torch.arange(Hv, device="cuda") // (Hv // case["Hk"])
    q, k, v = s["q"].double()[:, :, head], s["k"].double()[:, :, head], s["v"].double()
    alpha, beta = s["g"].double().exp(), s["beta"].double()
    S = torch.zeros(B, Hv, Dk, Dv, device="cuda", dtype=torch.float64) if s["state"] is None else s["state"].double()
    out = s["out"].double()
    steps = _lengths(case) if case["op"] == "clip" else [T if a else 0 for a in _active(case)]
    steps = torch.tensor(steps, device="cuda")
    ragged = case.get("ragged") or case.get("masked")
    for t in range(T):                     # the definition, frame by frame
        aS = alpha[:, t, :, None, None] * S
        e = beta[:, t, :, None, None] * (v[:, t, :, None] - k[:, t, :, None] @ aS)
        new = torch.baddbmm(aS.flatten(0, 1), k[:, t, :, :, None].flatten(0, 1), e.flatten(0, 1)).view_as(aS)
        o = (q[:, t, :, None] @ new).squeeze(2) / math.sqrt(Dk)
        if ragged:
            on = (t < steps)[:, None, None]
            S, out[:, t] = torch.where(on[..., None], new, S), torch.where(on, o, out[:, t])
        else:
            S, out[:, t] = new, o
    return out, S
