#!/usr/bin/env python3
"""bench.py -- throughput of the DPDFNet enhancement hot path on MI355X.

    python bench.py --gpus N --steps K --warmup W

A "step" is one pass of the whole offline hot path (`dpdf_enhance_batch`: centre/reflect STFT ->
frame function over every frame -> attenuation-limit -> iSTFT/OLA/alignment) over one batch of
synthetic clips per GPU, inputs and outputs resident in HBM.  Workload = BASELINE.json's metric
configuration: dpdfnet4 @ 16 kHz, 256 clips x 10 s per GPU (configs[2] is 2048 clips over 8 GPUs
= 256 per GPU, so per-GPU work is fixed: weak scaling).  One process per GPU; for N > 1 the driver
launches this file under torch.distributed.run and the enhanced PCM of every rank is gathered to
rank 0 over RCCL inside the timed region (the only collective on the path).

Rank 0 prints ONE JSON line with the contract fields plus `value_incl_pcie` (the same steps including
the H2D / D2H of the PCM), `roofline` (dominant kernel, measured with HIP events on the
engine's own streams in a pass of the same steps right after the timed region) and `cpu_baseline` (the CPU
oracle -- a port of the reference's frame-at-a-time execution model -- timed on the host cores on
a bounded sample; the reference's own CPU runtime, onnxruntime + downloaded .onnx files, is not
available offline).
"""
from __future__ import annotations

import argparse
import json
import os
import signal
import subprocess
import sys
import threading
import time
from pathlib import Path

import numpy as np

_PROC_T0 = time.perf_counter()
ROOT = Path(__file__).resolve().parent
sys.path.insert(0, str(ROOT))
os.environ.setdefault("GPU_MAX_HW_QUEUES", "8")      # before torch / HIP initialise: see dpdfnet_amd/__init__.py

METRIC = "frames/s (10 ms hop) per MI355X, dpdfnet4@16 kHz; PESQ Δ vs ref ≤0.001"
MODEL, SR, NB = "dpdfnet4", 16000, 4
CLIP_SECONDS = 10.0
WEIGHT_SEED = 20260417
FP32_MFMA_PEAK_TFLOPS = 157.3          # /opt/skills/guides/MI355X_MICROARCH.md: v_mfma_f32_16x16x4_f32 dense peak
BF16_MFMA_PEAK_TFLOPS = 2500.0         # ... dense bf16 peak (~2.5 PF; the guide measured >= 2382): what the limb kernels' MFMAs are priced against
LIMB_TERMS = 6                         # bf16 MFMAs per fp32 product term in gru_limb.h (3 x 3 limbs, the three products below 2^-24 dropped)
GRU64_FLOP_PER_ROW_STEP = 2 * 3 * 64 * (64 + 64)   # r,z,n gates x 64 units x (W_ih x + W_hh h), MAC = 2 FLOP
FLOP_PER_FRAME = 45.18e6               # algorithmic FLOP / frame, dpdfnet4
# SURVEY.md 8(d), measured with forward hooks on the reference modules: algorithmic MFLOP / frame of every registry model
FLOP_PER_FRAME_BY_MODEL = {(16000, 0): 6.64e6, (16000, 2): 25.91e6, (16000, 4): 45.18e6, (16000, 8): 83.71e6,
                           (48000, 2): 45.68e6, (48000, 8): 136.51e6}


def synth_clips(n_clips: int, n: int, sr: int, first_seed: int) -> np.ndarray:
    """x = 0.05 N(0,1) + 0.1 sin(2 pi f0 t)(1 + sin(2 pi 3 t)), f0 ~ U[100,1000] Hz."""
    t = np.arange(n, dtype=np.float32) / np.float32(sr)
    out = np.empty((n_clips, n), dtype=np.float32)
    for i in range(n_clips):
        rng = np.random.default_rng(first_seed + i)
        f0 = np.float32(rng.uniform(100.0, 1000.0))
        x = 0.05 * rng.standard_normal(n, dtype=np.float32)
        x += np.float32(0.1) * np.sin(np.float32(2 * np.pi) * f0 * t) * (1.0 + np.sin(np.float32(2 * np.pi * 3.0) * t))
        out[i] = np.clip(x, -1.0, 1.0)
    return out


def banked_trace(kind: str) -> str:
    """profiles/r<N>_<kind>_kernel_stats.csv of the latest round banked under profiles/ (tools/bank_profiles.sh), by name."""
    import re
    best, best_n = f"profiles/rN_{kind}_kernel_stats.csv (none banked)", -1
    for f in (ROOT / "profiles").glob(f"r*_{kind}_kernel_stats.csv"):
        mt = re.fullmatch(rf"r(\d+)_{kind}_kernel_stats\.csv", f.name)          # (not r5_limbs_pipelined_... for "pipelined")
        if mt and int(mt.group(1)) > best_n:
            best, best_n = f"profiles/{f.name}", int(mt.group(1))
    return best


def usable_cores() -> int:
    """Cores this process may actually use: affinity mask capped by the cgroup CPU quota (the GPU
    box exposes 256 hardware threads but cpu.max limits the container to a few of them)."""
    n = len(os.sched_getaffinity(0)) if hasattr(os, "sched_getaffinity") else (os.cpu_count() or 1)
    try:
        quota, period = Path("/sys/fs/cgroup/cpu.max").read_text().split()[:2]
        if quota != "max":
            n = min(n, max(1, int(int(quota) / int(period))))
    except (OSError, ValueError):
        try:
            q = int(Path("/sys/fs/cgroup/cpu/cpu.cfs_quota_us").read_text())
            p_ = int(Path("/sys/fs/cgroup/cpu/cpu.cfs_period_us").read_text())
            if q > 0:
                n = min(n, max(1, q // p_))
        except (OSError, ValueError):
            pass
    return max(1, n)


def cpu_baseline(blob: np.ndarray, seconds_per_clip: float, clips_per_thread: int) -> dict:
    """Time the CPU oracle (oracle/dpdf_oracle.c) the way the reference runs: one clip per thread,
    frame at a time, batch 1 (reference package/src/dpdfnet/cli.py:249-259)."""
    from oracle import oracle as orc
    cores = usable_cores()
    n = int(seconds_per_clip * SR)
    clips = synth_clips(cores * clips_per_thread, n, SR, 99000)
    oracles = [orc.Oracle(SR, NB, blob) for _ in range(cores)]
    frames = oracles[0].num_frames(n)

    def work(i: int) -> None:
        for j in range(clips_per_thread):
            oracles[i].enhance(clips[i * clips_per_thread + j])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(cores)]
    t0 = time.perf_counter()
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    dt = time.perf_counter() - t0
    total = cores * clips_per_thread * frames
    return {
        "value": total / dt, "unit": "frames/s", "cores": cores, "kind": "port", "host_threads_visible": os.cpu_count(),
        "sample": f"{cores * clips_per_thread} clips x {seconds_per_clip:g} s ({total} frames), one clip per thread, "
                  f"oracle/dpdf_oracle.c fp32 frame-at-a-time; {dt:.1f} s wall",
        "ms_per_frame_per_thread": 1e3 * dt / (clips_per_thread * frames),
    }


def parity_vs_oracle(blob: np.ndarray, wav_host: np.ndarray, out_host: np.ndarray, slots, clip_seed0=None) -> dict:
    """The timed step's OWN output (automatic chunk schedule, the execution shape `value` is measured on) against the CPU
    oracle on the same clips: a few slots of the batch, one oracle clip per thread, OUTSIDE the timed region.  The oracle is
    the checker here, never the thing measured (reference package/src/dpdfnet/api.py:51-113 is what both restate)."""
    from oracle import oracle as orc
    errs, sig = {}, {}

    stoi, sisnr = {}, {}

    def work(b: int) -> None:
        ref = orc.Oracle(SR, NB, blob).enhance(wav_host[b])
        errs[b] = float(np.sqrt(np.mean((out_host[b].astype(np.float64) - ref) ** 2)))
        sig[b] = float(np.sqrt(np.mean(ref.astype(np.float64) ** 2)))
        # north_star: "PESQ/STOI identical to 3 d.p."  pesq / pystoi are absent here; evalkit.stoi_np restates STOI from its paper (unpinned
        # against pystoi, and says so) -- the SAME function on both outputs against the clip's clean component, plus SI-SNR of ours vs the oracle
        try:
            from dpdfnet_amd.evalkit import si_snr, stoi_np
            rng = np.random.default_rng(clip_seed0 + b) if clip_seed0 is not None else None
            if rng is not None:
                n = wav_host.shape[1]
                t = np.arange(n, dtype=np.float32) / np.float32(SR)
                f0 = np.float32(rng.uniform(100.0, 1000.0))
                clean = np.float32(0.1) * np.sin(np.float32(2 * np.pi) * f0 * t) * (1.0 + np.sin(np.float32(2 * np.pi * 3.0) * t))
                stoi[b] = (round(float(stoi_np(clean, out_host[b], SR)), 4), round(float(stoi_np(clean, ref, SR)), 4))
            sisnr[b] = round(float(si_snr(ref, out_host[b])), 1)
        except Exception as e:          # (metrics are a courtesy here; the RMS check above is the gate)
            stoi[b] = f"{type(e).__name__}: {e}"

    ths = [threading.Thread(target=work, args=(int(b),)) for b in slots]
    for th in ths:
        th.start()
    for th in ths:
        th.join()
    tol = 2e-6
    return {"rms_max": max(errs.values()), "clips": [int(b) for b in slots], "rms_per_clip": [errs[int(b)] for b in slots],
            "signal_rms": [sig[int(b)] for b in slots], "tol": tol, "ok": bool(max(errs.values()) < tol),
            "stoi_np_ours_vs_oracle_output": [stoi.get(int(b)) for b in slots], "si_snr_db_ours_against_oracle": [sisnr.get(int(b)) for b in slots],
            "metrics_note": "STOI of our output and of the oracle's output against the clip's clean component with evalkit.stoi_np (a restatement of the STOI paper, "
                            "NOT pinned against pystoi, which like pesq is absent here): the pair must agree to 3 d.p.; SI-SNR as the reference's script computes it",
            "against": "oracle/dpdf_oracle.c (pinned to the reference's goldens) on the same clips; output of the LAST timed step"}


def sparse_stream_parity(m, st, sr_: int, nb_: int, S: int, hops: int = 60) -> dict:
    """configs[4] on spectrally SPARSE input: the 48 kHz features are 10 log10(|X| + 1e-10) per bin, so bins
    that hold nothing but the analysis transform's rounding residue become -60 dB features that differ between STFT
    implementations.  All S streams of the timed engine are reset and fed, hop by hop through the same C-ABI call the timing used,
    band-limited (< 6 kHz) float32 noise, the same as 16-bit PCM, and 0.25 s of silence followed by that signal (classes cycling
    over the streams); streams 0..2 are compared with the oracle's StreamEnhancer restatement (float64 rfft of the float32 frame,
    the shipped reference's arithmetic under its numpy pin: package/src/dpdfnet/stream.py:119-126), AFTER the timed region."""
    from oracle import oracle as orc
    from dpdfnet_amd import backend
    from dpdfnet_amd.weights import synth_blob
    hop = m.hop
    n = hops * hop
    rng = np.random.default_rng(48)
    spec = np.fft.rfft(rng.standard_normal(n))
    spec[np.fft.rfftfreq(n, 1.0 / sr_) > 6000.0] = 0.0
    bl = np.fft.irfft(spec, n)
    bl = (0.14 * bl / np.sqrt(np.mean(bl ** 2))).astype(np.float32)
    classes = {"bl_f32": bl, "bl_i16": (np.round(bl * 32768.0) / 32768.0).astype(np.float32),
               "sil_sig": np.concatenate([np.zeros(sr_ // 4, np.float32), bl[: n - sr_ // 4]])}
    names = list(classes)
    rows = np.stack([classes[names[i % 3]] for i in range(S)])
    st.reset()
    st.prime(rows[:, :hop].copy())
    got = np.concatenate([st.process(rows[:, j * hop:(j + 1) * hop].copy()) for j in range(1, hops)], axis=1)
    blob = synth_blob(backend.manifest(sr_, nb_), WEIGHT_SEED)
    errs = {}

    def work(i: int) -> None:
        ref = orc.Oracle(sr_, nb_, blob).stream(rows[i])
        errs[names[i]] = float(np.sqrt(np.mean((got[i].astype(np.float64) - ref[: got.shape[1]]) ** 2)))

    ths = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for th in ths:
        th.start()
    for th in ths:
        th.join()
    same = all(np.array_equal(got[i], got[i % 3]) for i in range(S))       # every stream of a class bit-identical to its first
    tol = 1e-5
    return {"rms_vs_oracle": {k: float(f"{v:.3g}") for k, v in errs.items()}, "signal_rms": 0.14, "hops": hops - 1, "tol": tol,
            "ok": bool(max(errs.values()) < tol and same), "streams_of_a_class_bit_identical": bool(same),
            "against": "oracle StreamEnhancer restatement (float64 analysis rfft of the float32 frame) hop by hop; north_star budget 1e-4"}


def ort_baseline(onnx_path: str, seconds: float = 15.0) -> dict:
    """OPTIONAL: the reference's own CPU runtime beside the GPU, when `onnxruntime` imports and DPDFNET_ONNX
    names a streaming dpdfnet4 .onnx file (neither exists in the offline image).  Session options are the reference's
    (package/src/dpdfnet/onnx_backend.py:21-49: one intra-op and one inter-op thread, ORT_ENABLE_ALL, CPUExecutionProvider);
    the loop is its per-frame session.run (api.py:96-104; onnx_model/infer_dpdfnet_onnx.py:299-306), one session per usable
    core, run for a bounded time on synthetic spectra."""
    import onnxruntime as ort  # noqa: F401  (ImportError is the caller's signal that the leg does not apply)
    opts = ort.SessionOptions()
    opts.intra_op_num_threads = 1
    opts.inter_op_num_threads = 1
    opts.graph_optimization_level = ort.GraphOptimizationLevel.ORT_ENABLE_ALL
    cores = usable_cores()
    sessions = [ort.InferenceSession(onnx_path, sess_options=opts, providers=["CPUExecutionProvider"]) for _ in range(cores)]
    s0 = sessions[0]
    ins, outs = s0.get_inputs(), s0.get_outputs()
    meta = s0.get_modelmeta().custom_metadata_map
    state0 = np.zeros(int(meta["state_size"]), dtype=np.float32)
    en = np.array([float(x) for x in meta["erb_norm_init"].split(",")], dtype=np.float32)
    sn = np.array([float(x) for x in meta["spec_norm_init"].split(",")], dtype=np.float32)
    state0[: en.size] = en
    state0[en.size: en.size + sn.size] = sn
    F = int(ins[0].shape[-2])
    rng = np.random.default_rng(1)
    spec = (0.1 * rng.standard_normal((64, 1, 1, F, 2))).astype(np.float32)
    counts = [0] * cores
    stop = time.perf_counter() + seconds

    def work(i: int) -> None:
        st = state0.copy()
        n = 0
        while time.perf_counter() < stop:
            _, st = sessions[i].run([outs[0].name, outs[1].name], {ins[0].name: spec[n & 63], ins[1].name: st})
            n += 1
        counts[i] = n

    ths = [threading.Thread(target=work, args=(i,)) for i in range(cores)]
    t0 = time.perf_counter()
    for th in ths:
        th.start()
    for th in ths:
        th.join()
    dt = time.perf_counter() - t0
    return {"value": sum(counts) / dt, "unit": "frames/s", "cores": cores, "kind": "ort",
            "sample": f"{sum(counts)} session.run calls (one frame each) over {dt:.1f} s, one 1-thread CPUExecutionProvider session per usable core, "
                      f"{Path(onnx_path).name}; options of package/src/dpdfnet/onnx_backend.py:21-49",
            "ms_per_frame_per_thread": 1e3 * dt * cores / max(1, sum(counts))}


def public_api_worker(B: int, steps: int, ref_path: str) -> None:
    """`bench.py --public-api-only`: the figure a USER of the package gets, in a process of its own (as a user's process is):
    `dpdfnet_amd.enhance_batch(list_of_numpy_clips, 16000, model="dpdfnet4")`, timed end to end per call (reference
    package/src/dpdfnet/api.py:51-113 is its per-clip counterpart): list of 1-D float32 arrays in, list of arrays out, everything
    in between (bucketing, the engine call on row pointers, H2D / D2H pipelined inside the library) inside the call."""
    import dpdfnet_amd
    N = int(CLIP_SECONDS * SR)
    clips = [c.copy() for c in synth_clips(B, N, SR, WEIGHT_SEED)]          # every clip in its own allocation, as a caller holds them
    kw = dict(model=MODEL, onnx_path=f"synthetic:{WEIGHT_SEED}")
    dpdfnet_amd.enhance_batch(clips, SR, **kw)                                # builds + caches the runtime, first-touch allocations
    t0 = time.perf_counter()
    outs = None
    for _ in range(steps):
        outs = dpdfnet_amd.enhance_batch(clips, SR, **kw)
    dt = (time.perf_counter() - t0) / steps
    T = 1 + (N + 320) // 160
    ref = dict(np.load(ref_path)) if ref_path and Path(ref_path).is_file() else {}
    res = {"value_public_api": B * T / dt, "ms_per_call": 1e3 * dt, "calls": steps,
           "call": f'dpdfnet_amd.enhance_batch(<list of {B} float32 arrays x {N} samples>, {SR}, model="{MODEL}")',
           "process": "own process (bench.py --public-api-only): a second engine handle in the bench process shares hardware queues "
                      "with the first one's streams and measures 4-5 % slower (docs/HISTORY.md section 3b)",
           "finite_output": bool(all(np.isfinite(o).all() for o in outs)),
           "max_abs_diff_vs_hbm_resident_output": (max(float(np.abs(outs[int(b)] - ref[b]).max()) for b in ref) if ref else None)}
    print("PUBLIC_API " + json.dumps(res), flush=True)


def public_api_pass(B: int, steps: int, ref_slots: dict, timeout_s: float = 600.0) -> dict:
    import subprocess
    import tempfile
    with tempfile.TemporaryDirectory() as td:
        ref_path = ""
        if ref_slots:
            ref_path = str(Path(td) / "ref_slots.npz")
            np.savez(ref_path, **{str(b): v for b, v in ref_slots.items()})
        r = subprocess.run([sys.executable, str(Path(__file__).resolve()), "--public-api-only", "--clips", str(B), "--steps", str(steps),
                            "--ref-slots", ref_path], capture_output=True, text=True, timeout=timeout_s, env=dict(os.environ))
    for l in r.stdout.splitlines():
        if l.startswith("PUBLIC_API "):
            return json.loads(l[len("PUBLIC_API "):])
    raise RuntimeError(f"no result line (rc {r.returncode}): {r.stderr[-300:]}")


def public_streams(model_name: str, sr_: int, S: int, calls: int = 200, pool_kw: dict = None) -> dict:
    """configs[4] through the objects a USER holds (reference package/src/dpdfnet/stream.py:74-165): (a) one
    `StreamEnhancer.group(S)` object, one hop of every stream per process() call; (b) S independent `pool.enhancer()` objects
    fed one hop each per round from four host threads (the pool coalesces the hops that arrive within its window into one
    device call).  Python staging, locks and the coalescing window are inside the figures."""
    import threading
    from dpdfnet_amd import StreamEnhancer, runtime as _rt
    kw = dict(model=model_name, onnx_path=f"synthetic:{WEIGHT_SEED}")
    hop = sr_ // 100
    rng = np.random.default_rng(1)
    pcm = (0.05 * rng.standard_normal((S, hop))).astype(np.float32)
    g = StreamEnhancer.group(S, **kw)
    g.process(np.concatenate([pcm, pcm], axis=1))          # window filled: primes, first hop
    for _ in range(20):
        g.process(pcm)
    t0 = time.perf_counter()
    for _ in range(calls):
        y = g.process(pcm)
    dt_group = (time.perf_counter() - t0) / calls
    assert y.shape == (S, hop)
    del g
    pool = StreamEnhancer.pool(S, **dict(dict(window_s=2e-4), **(pool_kw or {})), **kw)
    members = [pool.enhancer() for _ in range(S)]
    pool.process_many([(m_, np.concatenate([pcm[i], pcm[i]])) for i, m_ in enumerate(members)])
    nthreads, rounds = 4, calls
    share = [list(range(t, S, nthreads)) for t in range(nthreads)]
    bar = threading.Barrier(nthreads + 1)

    def feeder(t: int) -> None:
        mine = [(members[i], pcm[i]) for i in share[t]]
        bar.wait()
        for _ in range(rounds):
            pool.process_many(mine)                         # this thread's streams: one request each, coalesced per round
        bar.wait()

    # (each thread hands its 16 streams to the pool together; the four threads' requests meet in the pool's round: the first
    # caller leads and fires as soon as every stream in use has queued, or after the window)
    ths = [threading.Thread(target=feeder, args=(t,)) for t in range(nthreads)]
    for th in ths:
        th.start()
    dc0 = pool.device_calls
    bar.wait(); t0 = time.perf_counter(); bar.wait()
    dt_pool = (time.perf_counter() - t0) / rounds
    for th in ths:
        th.join()
    calls_per_round = (pool.device_calls - dc0) / rounds
    # the same pattern with NATIVE feeder threads (tools/pool_native_feeders.cpp: four std::threads, each submitting its 16 streams'
    # hops through dpdf_streams_submit_block): what the library's pool costs without CPython's GIL hand-offs between the feeders
    native = {}
    try:
        import ctypes
        helper = ctypes.CDLL(str(Path(__file__).resolve().parent / "tools" / "libpool_native_feeders.so"))
        L = pool._streams.model._L
        us = ctypes.c_double(0.0)
        dc1 = pool.device_calls
        helper.pool_native_feeders.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                               ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_double)]
        fn = ctypes.cast(L.dpdf_streams_submit_block, ctypes.c_void_p)
        for _ in range(2):      # (first pass: thread start-up, buffers)
            rc = helper.pool_native_feeders(pool._streams._h, fn, S, nthreads, rounds, hop, pcm.ctypes.data, None, ctypes.byref(us))
        native = {"us_per_round_native_feeders_4_threads": round(us.value, 1), "native_feeder_failures": int(rc),
                  "native_device_calls_per_round": round((pool.device_calls - dc1) / (2 * rounds), 2)}
    except OSError as e:
        native = {"native_feeders": f"helper not built ({e})"}
    for m_ in members:
        m_.close()
    del pool, members
    _rt.clear_cache()
    return {"us_per_call_public_group": round(1e6 * dt_group, 1),
            "us_per_round_public_pool_4_threads": round(1e6 * dt_pool, 1), "pool_device_calls_per_round": round(calls_per_round, 2), **native,
            "note": "group: StreamEnhancer.group(S).process([S, hop]) per hop; pool: S pool.enhancer() objects, four host threads "
                    "each feeding its 16 members one hop per round through process_many(); the pool coalesces the four threads' requests into one "
                    "device call per round (the round fires when all 64 streams in use have queued; it waits at most 2 ms for streams that rode in "
                    "the previous round, 200 us for the others); native feeders: the same four-thread pattern from std::threads on the C ABI "
                    "(tools/pool_native_feeders.cpp) -- the pool's own cost; the difference to the Python threads is CPython (GIL hand-offs "
                    "between the four feeders + ~20 us of interpreter per process_many call)"}



def public_streams_pass(model_name: str, sr_: int, S: int, timeout_s: float = 600.0) -> dict:
    """`public_streams` in a process of its own (bench.py --public-streams-only): like the public batch API it is what a user's process
    does, and further engine handles in THIS process would share hardware queues with the ones measured before and after."""
    import subprocess
    r = subprocess.run([sys.executable, str(Path(__file__).resolve()), "--public-streams-only", f"{model_name},{sr_},{S}"],
                       capture_output=True, text=True, timeout=timeout_s, env=dict(os.environ))
    for l in r.stdout.splitlines():
        if l.startswith("PUBLIC_STREAMS "):
            return json.loads(l[len("PUBLIC_STREAMS "):])
    raise RuntimeError(f"no result line (rc {r.returncode}): {r.stderr[-300:]}")


def other_configs(only=None) -> dict:
    """BASELINE.json's remaining single-GPU configurations, timed briefly beside the headline (they are parity-test
    cases in tests/test_gpu_fullsize.py; these are their speeds): dpdfnet2 / dpdfnet8 at 256 clips x 10 s, one clip
    through the engine (what a single `enhance()` call costs), and configs[4]: 64 concurrent device-resident
    dpdfnet8_48khz_hr streams, one 10 ms hop per call (host PCM in, host PCM out)."""
    import torch
    from dpdfnet_amd import backend
    from dpdfnet_amd.weights import synth_blob
    out: dict = {}
    n = int(CLIP_SECONDS * SR)

    def offline(nb: int, B: int, reps: int, **opts) -> float:
        m = backend.HipModel(SR, nb, synth_blob(backend.manifest(SR, nb), WEIGHT_SEED), device=torch.cuda.current_device())
        for k, v in opts.items():
            m.set_option(k, v)
        wav = torch.from_numpy(synth_clips(min(B, 8), n, SR, 5000)).cuda().repeat((B + 7) // 8, 1)[:B].contiguous()
        y = torch.empty_like(wav)
        m.enhance_batch_device(wav.data_ptr(), B, n, y.data_ptr(), None); m.sync()
        t0 = time.perf_counter()
        for _ in range(reps):
            m.enhance_batch_device(wav.data_ptr(), B, n, y.data_ptr(), None)
        m.sync()
        dt = (time.perf_counter() - t0) / reps
        T = m.num_frames(n); rec = m.recovery_count; m.close()
        return B * T / dt, 1e3 * dt, rec

    def mfma(fps: float, sr: int, nb: int) -> float:
        return round(fps * FLOP_PER_FRAME_BY_MODEL[(sr, nb)] / 1e12 / FP32_MFMA_PEAK_TFLOPS, 4)

    def streams(sr_: int, nb_: int, S: int, calls: int = 200) -> dict:
        m = backend.HipModel(sr_, nb_, synth_blob(backend.manifest(sr_, nb_), WEIGHT_SEED), device=torch.cuda.current_device())
        st = backend.HipStreams(m, S)
        rng = np.random.default_rng(0)
        hop = m.hop
        st.prime((0.05 * rng.standard_normal((S, hop))).astype(np.float32))
        pcm = (0.05 * rng.standard_normal((S, hop))).astype(np.float32)
        for _ in range(20):
            st.process(pcm)
        t0 = time.perf_counter()
        for _ in range(calls):
            st.process(pcm)
        dt = (time.perf_counter() - t0) / calls
        # the same hops from a native loop (tools/pool_native_feeders.cpp: native_hop_loop calls dpdf_streams_process `calls` times): the C-ABI
        # figure without the interpreter between the hops
        native_us = None
        try:
            import ctypes
            helper = ctypes.CDLL(str(Path(__file__).resolve().parent / "tools" / "libpool_native_feeders.so"))
            helper.native_hop_loop.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p,
                                               ctypes.c_int, ctypes.POINTER(ctypes.c_double)]
            us = ctypes.c_double(0.0)
            outb = np.empty_like(pcm)
            fn = ctypes.cast(m._L.dpdf_streams_process, ctypes.c_void_p)
            if helper.native_hop_loop(st._h, fn, calls, 20, pcm.ctypes.data, outb.ctypes.data, backend.DPDF_HOST_PTRS, ctypes.byref(us)) == 0:
                native_us = round(us.value, 1)
        except (OSError, AttributeError):
            pass
        sparse = sparse_stream_parity(m, st, sr_, nb_, S) if sr_ == 48000 else None
        rec = m.recovery_count
        st.close(); m.close()
        d = backend.query_dims(sr_, nb_)
        # Latency model of a hop (docs/HISTORY.md section 4): the two branches run side by side, each a chain of nb x (F' dependent
        # GRU-64 steps + one glue launch); the DF branch (F' = 48) is the longer one.  Measured minima on this chip
        # (tools/scan4_bench.hip, rocprofv3 traces of single hops, profiles/r*_stream_hop_*): 0.41 us per 4-row scan step (64 x
        # 8.4-cycle v_mfma_f32_4x4x1 + one LDS round trip + the gate chain; 0.55 until round 4), ~1.5 us per dependent kernel boundary.
        # Launches on the chain of a one-chunk call (main stream; the decoders one after the other): prologue / import, STFT,
        # features, encoder front end (+ projection at 48 kHz x 64), nb x (scan + glue in one launch, dprnn_hop_block.h), emb_in,
        # 5 GRU-256 steps, emb_out, df_out, pathway conv, dec_in, decoder pyramid, mask + deep filter, iSTFT, overlap-add = nb + 19
        # (2 nb + 19 until round 4, 2 nb + 30 in round 3).
        steps = nb_ * d.Fd
        chain = nb_ + 19
        bound_us = steps * 0.41 + chain * 1.5
        return {"us_per_call": round(1e6 * dt, 1), "us_per_call_native_loop": native_us, "frames_per_s": round(S / dt), "rtf": round(dt / (hop / sr_), 4),
                "mfma_frac": mfma(S / dt, sr_, nb_),
                "latency_model": {"dependent_gru64_steps": steps, "dependent_launches_on_critical_path": chain,
                                  "bound_us": round(bound_us, 1), "achieved_over_bound": round(1e6 * dt / bound_us, 2)},
                "io": "host PCM in, host PCM out (pinned staging, zero-copy), one device call per hop", "recovery_count": rec,
                **({"parity_sparse": sparse} if sparse else {})}

    # Every side configuration is measured in a process of its own (`bench.py --side-config <name>`): engine handles created
    # one after the other in ONE process end up sharing hardware queues (docs/HISTORY.md section 3b) -- the fifth handle of the bench
    # process measured dpdfnet8 at 194.7 ms per step, a fresh process 187.0.
    if only == "one_clip":
        fps, ms, rec = offline(NB, 1, 5)
        return {"frames_per_s": round(fps), "ms_per_call": round(ms, 2), "rtf": round(ms / 1e3 / CLIP_SECONDS, 5), "recovery_count": rec}
    if only == "streams48":
        return streams(48000, 8, 64)
    if only == "streams16":
        return streams(16000, 2, 1)                                            # one StreamEnhancer (the reference's unit of work)
    if only in ("offline2", "offline8"):
        nb = int(only[-1])
        fps, ms, rec = offline(nb, 256, 3)
        return {"frames_per_s": round(fps), "ms_per_step": round(ms, 2), "whole_path_over_fp32_peak": mfma(fps, SR, nb), "recovery_count": rec}
    if only == "offline48_2":                                                  # dpdfnet2_48khz_hr, 256 clips x 10 s (the 48 kHz family offline)
        n48 = int(CLIP_SECONDS * 48000)
        m = backend.HipModel(48000, 2, synth_blob(backend.manifest(48000, 2), WEIGHT_SEED), device=torch.cuda.current_device())
        wav = torch.from_numpy(synth_clips(8, n48, 48000, 5000)).cuda().repeat(32, 1).contiguous()
        y = torch.empty_like(wav)
        m.enhance_batch_device(wav.data_ptr(), 256, n48, y.data_ptr(), None); m.sync()
        t0 = time.perf_counter()
        for _ in range(3):
            m.enhance_batch_device(wav.data_ptr(), 256, n48, y.data_ptr(), None)
        m.sync()
        dt = (time.perf_counter() - t0) / 3
        fps = 256 * m.num_frames(n48) / dt
        rec = m.recovery_count; m.close()
        return {"frames_per_s": round(fps), "ms_per_step": round(1e3 * dt, 2), "whole_path_over_fp32_peak": mfma(fps, 48000, 2), "recovery_count": rec}
    if only == "public_streams48":
        return public_streams("dpdfnet8_48khz_hr", 48000, 64)
    if only is not None:
        raise SystemExit(f"unknown side configuration {only!r}")

    # ONE child process for all of them (`bench.py --side-config all`): it imports torch and the package once -- on a cold box the
    # imports are most of a fresh process's time -- and then FORKS one worker per configuration before anything has touched the
    # GPU, so that every configuration still runs in a process with no other engine handle and no HIP state of its predecessors.
    rc, so, se = run_child_streaming([sys.executable, str(Path(__file__).resolve()), "--side-config", "all"], 600.0, dict(os.environ))
    res = None
    for l in so.splitlines():
        if l.startswith("SIDE "):
            res = json.loads(l[len("SIDE "):])
    if res is None:
        return {"error": f"no result line from the side-configuration process (rc {rc}): {se[-300:]}"}
    out[f"{MODEL}_16k_1x10s"] = res["one_clip"]
    s48 = res["streams48"]
    pub = res["public_streams48"]
    if "error" not in pub and "us_per_call" in s48:
        pub["public_group_over_c_abi"] = round(pub["us_per_call_public_group"] / s48["us_per_call"], 3)
        pub["public_pool_over_c_abi"] = round(pub["us_per_round_public_pool_4_threads"] / s48["us_per_call"], 3)
        if "us_per_round_native_feeders_4_threads" in pub:
            pub["native_pool_over_c_abi"] = round(pub["us_per_round_native_feeders_4_threads"] / s48["us_per_call"], 3)
    s48["public_objects"] = pub
    out["dpdfnet8_48khz_hr_64_streams_1_hop"] = s48
    out["dpdfnet2_16k_1_stream_1_hop"] = res["streams16"]
    for nb in (2, 8):
        out[f"dpdfnet{nb}_16k_256x10s"] = res[f"offline{nb}"]
    out["dpdfnet2_48khz_hr_256x10s"] = res["offline48_2"]
    out["side_process"] = res.get("_timing")
    return out


SIDE_ORDER = ("one_clip", "streams48", "public_streams48", "streams16", "offline2", "offline8", "offline48_2")


def side_all() -> dict:
    """`bench.py --side-config all`: torch, numpy and the package imported ONCE, no GPU call made; then one fork per configuration
    (latency-bound ones first).  The fork child runs `other_configs(name)` in a process that has never initialised HIP, writes its
    JSON to a pipe and leaves with os._exit; a configuration that overruns 240 s is killed -- that exact pid -- and reported."""
    import select
    import signal
    import torch  # noqa: F401   (imported, not initialised: torch.cuda is lazy)
    import dpdfnet_amd  # noqa: F401
    from dpdfnet_amd import backend, weights  # noqa: F401
    res, timing = {}, {"imports_s": round(time.perf_counter() - _PROC_T0, 2)}
    for name in SIDE_ORDER:
        t0 = time.perf_counter()
        r, w = os.pipe()
        pid = os.fork()
        if pid == 0:
            os.close(r)
            try:
                torch.cuda.set_device(0)
                payload = other_configs(name)
            except BaseException as exc:      # the parent must always get a line
                payload = {"error": f"{type(exc).__name__}: {exc}"[:300]}
            try:
                os.write(w, json.dumps(payload).encode())
            finally:
                os._exit(0)
        os.close(w)
        data, deadline = b"", time.perf_counter() + 240.0
        while True:
            left = deadline - time.perf_counter()
            if left <= 0:
                os.kill(pid, signal.SIGKILL)
                data = json.dumps({"error": "timed out after 240 s"}).encode()
                break
            if select.select([r], [], [], min(left, 1.0))[0]:
                chunk = os.read(r, 1 << 16)
                if not chunk:
                    break
                data += chunk
        os.close(r)
        os.waitpid(pid, 0)
        try:
            res[name] = json.loads(data.decode()) if data else {"error": "the worker wrote nothing"}
        except ValueError:
            res[name] = {"error": f"unparsable worker output: {data[:200]!r}"}
        timing[name + "_s"] = round(time.perf_counter() - t0, 2)
    res["_timing"] = timing
    return res


def _free_port() -> int:
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def self_launch(n: int) -> int:
    """`python bench.py --gpus N` invoked PLAINLY (no launcher, no WORLD_SIZE in the environment): start the N ranks
    ourselves -- the same `torch.distributed.run` command line the driver uses, one process per GPU on this node,
    rendezvous on 127.0.0.1 -- and pass the ranks' stdout / stderr through, so that either launch style gives the one
    JSON line from rank 0.  (The reference's counterpart is one host thread per file, cli.py:249-259, 308-311.)"""
    import subprocess
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", DPDF_BENCH_SELF_LAUNCHED="1")
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")          # dmabuf IPC only on these hosts (RCCL p2p needs it)
    env.setdefault("OMP_NUM_THREADS", "1")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", str(n),
           "--master-addr", "127.0.0.1", "--master-port", str(_free_port()), str(Path(__file__).resolve())] + sys.argv[1:]
    print(f"[bench.py] --gpus {n} without a launcher: starting {n} ranks with torch.distributed.run", file=sys.stderr, flush=True)
    return subprocess.run(cmd, env=env).returncode


def _stamp(stage: str) -> None:
    """One line per stage on stderr, flushed as it happens: what a parent that has to give up on this process still holds."""
    print(f"STAGE {time.perf_counter() - _PROC_T0:8.2f}s {stage}", file=sys.stderr, flush=True)


def dist_selftest_worker() -> None:
    """`bench.py --dist-selftest-only`: one rank, backend nccl (= RCCL on ROCm): communicator init bound to the device, the
    collectives the N > 1 path of this file uses (all_reduce MAX on a device tensor = the max-over-ranks clock, barrier,
    all_gather_object, a grouped isend/irecv = gather_to_root's launch shape) -- so that RCCL has executed this code's
    calls on the box even where only one GPU is leased.  Every stage is stamped on stderr BEFORE it starts (the parent keeps
    the stamps when it has to kill this process: `hung_at`); prints one JSON object on stdout."""
    import datetime
    _stamp("import torch")
    import torch
    import torch.distributed as dist
    res = {"backend": "nccl (RCCL)", "world_size": 1}
    if os.environ.get("DPDF_BENCH_FAKE_RCCL_HANG") == "1":       # test hook: a communicator init that never returns
        _stamp("init_process_group(nccl) [DPDF_BENCH_FAKE_RCCL_HANG=1: sleeping instead]")
        time.sleep(3600)
    t0 = time.perf_counter()
    try:
        os.environ["MASTER_ADDR"] = "127.0.0.1"
        os.environ["MASTER_PORT"] = str(_free_port())
        os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
        _stamp("torch.cuda.set_device(0)")
        torch.cuda.set_device(0)
        _stamp("first device touch (torch.zeros on cuda:0)")
        torch.zeros(1, device="cuda"); torch.cuda.synchronize()
        res["device_up_ms"] = round(1e3 * (time.perf_counter() - t0), 1)
        _stamp("init_process_group(nccl, world_size=1, device_id=cuda:0)")
        t1 = time.perf_counter()
        dist.init_process_group(backend="nccl", rank=0, world_size=1, device_id=torch.device("cuda", 0),
                                timeout=datetime.timedelta(seconds=45))
        res["init_ms"] = round(1e3 * (time.perf_counter() - t1), 1)
        t = torch.tensor([1.25], dtype=torch.float64, device="cuda")
        _stamp("all_reduce(MAX)")
        t1 = time.perf_counter()
        dist.all_reduce(t, op=dist.ReduceOp.MAX); torch.cuda.synchronize()
        res["first_all_reduce_ms"] = round(1e3 * (time.perf_counter() - t1), 1)
        res["all_reduce_ok"] = bool(float(t.item()) == 1.25)
        _stamp("barrier")
        dist.barrier(); torch.cuda.synchronize()
        res["barrier_ok"] = True
        _stamp("all_gather_object")
        objs = [None]
        dist.all_gather_object(objs, {"rank": 0})
        res["all_gather_object_ok"] = objs == [{"rank": 0}]
        try:
            ver = torch.cuda.nccl.version()
            res["rccl_version"] = ".".join(str(v) for v in ver) if isinstance(ver, tuple) else str(ver)
        except Exception:
            pass
        try:        # gather_to_root's launch shape (one grouped isend + irecv), rank 0 to itself
            _stamp("batch_isend_irecv (self)")
            a = torch.arange(1 << 20, dtype=torch.float32, device="cuda"); b = torch.zeros_like(a)
            for q in dist.batch_isend_irecv([dist.P2POp(dist.irecv, b, 0), dist.P2POp(dist.isend, a, 0)]):
                q.wait()
            torch.cuda.synchronize()
            res["grouped_p2p_self_ok"] = bool(torch.equal(a, b))
        except Exception as exc:
            res["grouped_p2p_self_ok"] = False
            res["grouped_p2p_self_error"] = f"{type(exc).__name__}: {exc}"[:200]
        _stamp("destroy_process_group")
        dist.destroy_process_group()
        res["rccl_init_ok"] = bool(res["all_reduce_ok"] and res["barrier_ok"] and res["all_gather_object_ok"])
    except Exception as exc:
        res["rccl_init_ok"] = False
        res["error"] = f"{type(exc).__name__}: {exc}"[:300]
    res["total_s"] = round(time.perf_counter() - _PROC_T0, 2)
    _stamp("done")
    print("DIST_SELFTEST " + json.dumps(res), flush=True)


def run_child_streaming(cmd, timeout_s: float, env=None):
    """Run `cmd`, collecting stdout and stderr AS THEY ARRIVE (reader threads), and kill it -- the exact process we started --
    at the deadline.  Returns (rc or None if killed, stdout, stderr): what a child printed before it hung is kept."""
    import subprocess
    p = subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, env=env, bufsize=1)
    bufs = {"out": [], "err": []}

    def pump(stream, key):
        for line in stream:
            bufs[key].append(line)

    ths = [threading.Thread(target=pump, args=(p.stdout, "out"), daemon=True), threading.Thread(target=pump, args=(p.stderr, "err"), daemon=True)]
    for th in ths:
        th.start()
    rc = None
    try:
        rc = p.wait(timeout=timeout_s)
    except subprocess.TimeoutExpired:
        p.kill()
        p.wait()
    for th in ths:
        th.join(timeout=5)
    return rc, "".join(bufs["out"]), "".join(bufs["err"])


def dist_selftest(timeout_s: float = 60.0) -> dict:
    """Run `dist_selftest_worker` in its OWN process under a deadline, with NCCL_DEBUG=INFO: a broken or hanging RCCL install is
    reported on the line with the stage it hung at and the tail of RCCL's own log, and can never take the headline measurement
    with it."""
    t0 = time.perf_counter()
    env = dict(os.environ, NCCL_DEBUG=os.environ.get("NCCL_DEBUG", "INFO"))
    try:
        rc, out, err = run_child_streaming([sys.executable, str(Path(__file__).resolve()), "--dist-selftest-only"], timeout_s, env)
    except Exception as exc:
        return {"rccl_init_ok": False, "error": f"{type(exc).__name__}: {exc}"[:300]}
    stages = [l[len("STAGE "):].strip() for l in err.splitlines() if l.startswith("STAGE ")]
    res = None
    for l in out.splitlines():
        if l.startswith("DIST_SELFTEST "):
            res = json.loads(l[len("DIST_SELFTEST "):])
    if res is None:
        log = "\n".join(l for l in (out + err).splitlines() if not l.startswith("STAGE "))
        res = {"rccl_init_ok": False,
               "error": (f"timed out after {timeout_s:g} s" if rc is None else f"no result line (rc {rc})"),
               "hung_at": stages[-1] if stages else "before the first stage (interpreter start-up)",
               "log_tail": log[-2048:]}
    res["stages"] = stages
    res["wall_s"] = round(time.perf_counter() - t0, 2)
    return res


_FALLBACK = threading.Lock()             # taken by the thread that falls back, for good: every other one waits for the process's end


def rerun_with_gloo_fallback(reason: str) -> None:
    """RCCL did not come up (or stopped answering) on this node: run the same command line on `--backend gloo --fallback-reason ...` as a child
    process and end with its exit code (a process that has initialised the GPU is not replaced by another program; the launcher that
    watches this rank sees nothing die).  Every rank gets here on its own -- by its watchdog, or by the exception RCCL raised -- and they
    meet again at a fresh TCP rendezvous one port above the launcher's.  The line then says `collective: "FALLBACK gloo: <reason>"`, the per-GPU compute figures are
    still measured, rc stays 0."""
    _FALLBACK.acquire()
    argv = [a for a in sys.argv[1:]]
    out, skip = [], False
    for a in argv:
        if skip:
            skip = False
            continue
        if a == "--backend":
            skip = True
            continue
        if a.startswith("--backend="):
            continue
        out.append(a)
    reason = " ".join(str(reason).split())[:300]
    env = dict(os.environ)
    env.setdefault("DPDF_BENCH_FALLBACK_PORT", str(int(env.get("MASTER_PORT", "29500")) + 17))
    print(f"[bench.py] rank {env.get('RANK', '0')}: RCCL unusable ({reason}); running again on --backend gloo (control plane + host-staged "
          f"gather), rendezvous 127.0.0.1:{env['DPDF_BENCH_FALLBACK_PORT']}", file=sys.stderr, flush=True)
    sys.stdout.flush()
    rc = 1
    try:
        rc = subprocess.call([sys.executable, str(Path(__file__).resolve())] + out + ["--backend", "gloo", "--fallback-reason", reason], env=env)
    finally:
        os._exit(rc if 0 <= rc < 256 else 1)      # the main thread may be stuck inside RCCL


class CollectiveWatchdog:
    """A hang inside RCCL (communicator init, a collective whose peer never arrives) raises nothing: a timer thread runs the
    rank again on the gloo fallback when the watched section overruns its deadline.  `stage()` names what is running (it goes on the
    line as the reason); `disarm()` ends the watch."""

    def __init__(self) -> None:
        self._timer = None
        self._stage = "(not started)"
        self._lock = threading.Lock()

    def stage(self, name: str) -> None:
        self._stage = name
        print(f"STAGE {time.perf_counter() - _PROC_T0:8.2f}s rank {os.environ.get('RANK', '0')}: {name}", file=sys.stderr, flush=True)

    def arm(self, seconds: float, stage: str) -> None:
        self.disarm()
        self.stage(stage)
        with self._lock:
            self._timer = threading.Timer(seconds, self._fire, args=(seconds,))
            self._timer.daemon = True
            self._timer.start()

    def disarm(self) -> None:
        with self._lock:
            if self._timer is not None:
                self._timer.cancel()
                self._timer = None
        with _FALLBACK:                  # an answer that comes once the fallback runs is too late
            pass

    def _fire(self, seconds: float) -> None:
        rerun_with_gloo_fallback(f"no answer within {seconds:g} s at stage `{self._stage}`")


def float64_recurrence_error() -> dict:
    """Both GRU-64 kernel families against a float64 recurrence on the same weights and inputs (tools/gru64_limb_bench: the carried state of
    the inter-band scan after 192 steps): the claim "the limb kernels are not narrower than fp32" as a number on the line."""
    exe = ROOT / "tools" / "gru64_limb_bench"
    if not exe.exists():
        return {"available": False, "why": "tools/gru64_limb_bench not built (__graft_entry__.build_tools)"}
    try:
        r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=180)
        import re
        m = re.search(r"float64 recurrence \((\d+) rows x (\d+) steps, state RMS ([0-9.e+-]+)\): fp32-MFMA kernel RMS ([0-9.e+-]+) max ([0-9.e+-]+) \| limb kernel RMS ([0-9.e+-]+) max ([0-9.e+-]+)", r.stdout)
        if not m:
            return {"available": False, "why": "no result line: " + (r.stdout + r.stderr)[-200:]}
        return {"available": True, "rows": int(m.group(1)), "steps": int(m.group(2)), "state_rms": float(m.group(3)),
                "fp32_mfma_kernels": {"rms": float(m.group(4)), "max": float(m.group(5))},
                "limb_kernels": {"rms": float(m.group(6)), "max": float(m.group(7))},
                "speed_isolated": [l.strip() for l in r.stdout.splitlines() if " x" in l and ("intra" in l or "inter (" in l)][:3]}
    except Exception as exc:
        return {"available": False, "why": f"{type(exc).__name__}: {exc}"[:200]}


def multi_gpu_summary(per_rank: list) -> dict:
    """What a first hardware scaling curve needs to be read without a re-run: the spread of the ranks' own step times and what the
    gather to rank 0 costs (device-side duration of the grouped receive on rank 0 -- it overlaps the next step's compute -- and as a
    fraction of the slowest rank's step)."""
    ms = [r["ms_per_step"] for r in per_rank if isinstance(r, dict)]
    if not ms:
        return {}
    root = next((r for r in per_rank if isinstance(r, dict) and r.get("rank") == 0), None)
    g = root.get("gather_device_ms_per_step") if root else None
    return {"per_rank_ms_min": min(ms), "per_rank_ms_max": max(ms), "per_rank_ms_spread": (max(ms) - min(ms)) / max(ms),
            "gather_ms_per_step_root_device": g, "gather_frac_of_step": (g / max(ms)) if g is not None else None,
            "gather_host_ms_per_step_max": max(r.get("gather_host_ms_per_step", 0.0) for r in per_rank if isinstance(r, dict))}


def main() -> None:
    if os.environ.get("DPDF_BENCH_TRACE_HANG"):          # debugging aid: every thread's Python stack on stderr after that many seconds
        import faulthandler
        faulthandler.dump_traceback_later(float(os.environ["DPDF_BENCH_TRACE_HANG"]), repeat=False, exit=False)
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=3)
    ap.add_argument("--warmup", type=int, default=1)
    ap.add_argument("--clips", type=int, default=256, help="clips per GPU")
    ap.add_argument("--chunk", type=int, default=int(os.environ.get("DPDF_CHUNK_FRAMES", "0")),
                    help="time-chunk length in frames (0 = engine default)")
    ap.add_argument("--overlap", type=int, default=-1, help="overlap bit mask (1 stage-2 stream, 2 ERB stream, 8 decoder fork, 16 8-/16-WG GRU-256 clusters; 0 serial; -1 engine default)")
    ap.add_argument("--no-fuse", action="store_true", help="run fc+LN of the DPRNN blocks as separate kernels")
    ap.add_argument("--fp32-mfma", action="store_true", help="A/B and traces only: time the fp32-MFMA GRU-64 kernels (gru64_limbs = 0, the default of rounds 1-5) as this run's mode; the line says so")
    ap.add_argument("--limbs", action="store_true", help="the default since round 6 (gru64_limbs = 3: the GRU-64 throughput kernels on bf16 limbs); kept so that older command lines still parse")
    ap.add_argument("--no-gather", action="store_true")
    ap.add_argument("--backend", default="nccl", help="torch.distributed backend (nccl = RCCL; gloo only to exercise the N>1 control flow on a box with fewer GPUs than ranks)")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-parity", action="store_true", help="skip the oracle check of the timed step's output (3 clips, a few seconds of CPU)")
    ap.add_argument("--no-isolated", action="store_true", help="skip the extra serial profiling step")
    ap.add_argument("--no-other-configs", action="store_true", help="skip the brief timings of BASELINE's other single-GPU configs")
    ap.add_argument("--no-pcie", action="store_true", help="skip the H2D/D2H-inclusive pass (value_incl_pcie)")
    ap.add_argument("--profile-steps", type=int, default=-1, help="steps of the per-kernel HIP-event pass after the timed region (-1 = --steps, 0 = none)")
    ap.add_argument("--opt", action="append", default=[], metavar="NAME=INT", help="engine A/B switch (dpdf_set_option), repeatable")
    ap.add_argument("--cpu-clip-seconds", type=float, default=10.0)
    ap.add_argument("--cpu-clips-per-thread", type=int, default=5)
    ap.add_argument("--dist-selftest", dest="dist_selftest", action="store_true", default=None,
                    help="N=1: also bring up a one-rank RCCL process group in a child process and run this file's collectives "
                         "on it (`rccl_selftest` / `rccl_init_ok` on the line); default on at N=1")
    ap.add_argument("--no-dist-selftest", dest="dist_selftest", action="store_false")
    ap.add_argument("--dist-selftest-only", action="store_true", help=argparse.SUPPRESS)
    ap.add_argument("--public-api-only", action="store_true", help=argparse.SUPPRESS)
    ap.add_argument("--ref-slots", default="", help=argparse.SUPPRESS)
    ap.add_argument("--public-streams-only", default="", help=argparse.SUPPRESS)
    ap.add_argument("--side-config", default="", help=argparse.SUPPRESS)
    ap.add_argument("--fallback-reason", default="", help=argparse.SUPPRESS)      # set by rerun_with_gloo_fallback
    args = ap.parse_args()
    if args.fallback_reason and sys.platform == "linux":
        import ctypes
        ctypes.CDLL(None).prctl(1, int(signal.SIGTERM), 0, 0, 0)        # PR_SET_PDEATHSIG: the launcher ends the rank that started this process

    if args.side_config == "all":
        print("SIDE " + json.dumps(side_all()), flush=True)
        return
    if args.side_config:
        import torch
        torch.cuda.set_device(0)
        print("SIDE " + json.dumps(other_configs(args.side_config)), flush=True)
        return

    if args.public_streams_only:
        name, sr_, S_ = args.public_streams_only.split(",")
        print("PUBLIC_STREAMS " + json.dumps(public_streams(name, int(sr_), int(S_))), flush=True)
        return

    if args.public_api_only:
        public_api_worker(args.clips, max(1, args.steps), args.ref_slots)
        return

    if args.dist_selftest_only:
        dist_selftest_worker()
        return
    if args.gpus > 1 and "WORLD_SIZE" not in os.environ:
        # plain `python bench.py --gpus N`: become the launcher (under torch.distributed.run WORLD_SIZE is set and we fall through)
        raise SystemExit(self_launch(args.gpus))

    timeline = {}
    marks = [time.perf_counter()]

    def mark(name: str) -> None:
        """Wall seconds of the phase that just ended (rides on the line as `timeline_s`: where a driver's clock around the run goes)."""
        now = time.perf_counter()
        timeline[name] = round(timeline.get(name, 0.0) + now - marks[0], 2)
        marks[0] = now

    timeline["interpreter_start_to_main"] = round(marks[0] - _PROC_T0, 2)
    import torch
    import torch.distributed as dist
    from dpdfnet_amd import backend
    from dpdfnet_amd.weights import synth_blob
    from dpdfnet_amd.multi_gpu import shard_range, gather_to_root
    mark("import_torch_and_engine")

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    if world != args.gpus:
        raise SystemExit(f"--gpus {args.gpus} but WORLD_SIZE={world}: launch with torch.distributed.run --nproc-per-node {args.gpus}")
    if not torch.cuda.is_available():
        raise SystemExit("bench.py needs a GPU (the HIP engine has no CPU fallback)")
    fake_hang = os.environ.get("DPDF_BENCH_FAKE_RCCL_HANG") == "1"      # test hook: RCCL's init never returns (exercises the fallback on one GPU)
    if args.backend != "nccl" or fake_hang:
        local_rank %= torch.cuda.device_count()      # functional test mode / fallback: ranks may share a GPU (on a full node they do not)
    elif local_rank >= torch.cuda.device_count():
        raise SystemExit(f"LOCAL_RANK {local_rank} but only {torch.cuda.device_count()} GPUs are visible: one rank per GPU")
    torch.cuda.set_device(local_rank)
    rccl_ranks = None
    wd = CollectiveWatchdog()
    wd_s = float(os.environ.get("DPDF_BENCH_RCCL_WATCHDOG_S", "120"))
    if world > 1:
        import datetime
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        if args.backend == "nccl":
            # communicator init + the first collectives under a watchdog: RCCL hangs raise nothing (round 4: a ONE-rank init sat
            # for 180 s on the driver's box); overrun or exception -> the rank runs again on the gloo fallback
            try:
                wd.arm(wd_s, "init_process_group(nccl, device_id)")
                if fake_hang:
                    time.sleep(3600)
                dist.init_process_group(backend="nccl", device_id=torch.device("cuda", local_rank),
                                        timeout=datetime.timedelta(seconds=wd_s + 60))
                wd.stage("pre-flight: all_reduce on the device")
                one = torch.ones(1, device="cuda")
                dist.all_reduce(one); torch.cuda.synchronize()
                if int(one.item()) != world:
                    raise RuntimeError(f"all_reduce of ones gave {one.item()} on {world} ranks")
                wd.stage("pre-flight: grouped point-to-point gather (4 MB per rank)")
                probe = torch.full((1, 1 << 20), float(rank), device="cuda")
                got = gather_to_root(probe, world, rank); torch.cuda.synchronize()
                if rank == 0 and [float(got[r, 0, 0]) for r in range(world)] != [float(r) for r in range(world)]:
                    raise RuntimeError("grouped p2p gather delivered the wrong rows")
                wd.stage("pre-flight: all_gather_object")
            except SystemExit:
                raise
            except Exception as exc:
                wd.disarm()
                rerun_with_gloo_fallback(f"{type(exc).__name__} at stage `{wd._stage}`: {exc}")
        elif args.fallback_reason:
            # an explicit store: under torch.distributed.run (TORCHELASTIC_USE_AGENT_STORE) a tcp:// init_method makes EVERY rank a
            # client of a store nobody hosts -- both ranks sat in the rendezvous for good (found by the fake-hang GPU test)
            store = dist.TCPStore("127.0.0.1", int(os.environ["DPDF_BENCH_FALLBACK_PORT"]), world, rank == 0,
                                  timeout=datetime.timedelta(seconds=120), wait_for_workers=True)
            dist.init_process_group(backend="gloo", store=store, rank=rank, world_size=world, timeout=datetime.timedelta(seconds=600))
        else:
            dist.init_process_group(backend=args.backend)
        # pre-flight: the process group really has N ranks and (under RCCL) every rank sits on its own GPU
        if dist.get_world_size() != args.gpus:
            raise SystemExit(f"process group has {dist.get_world_size()} ranks, --gpus says {args.gpus}")
        props = torch.cuda.get_device_properties(local_rank)
        me = {"rank": rank, "device": torch.cuda.current_device(), "uuid": str(getattr(props, "uuid", "")), "name": props.name}
        everyone = [None] * world
        dist.all_gather_object(everyone, me)
        rccl_ranks = sorted(everyone, key=lambda r: r["rank"])
        if args.backend == "nccl":
            devs = [(r["device"], r["uuid"]) for r in rccl_ranks]
            if len(set(devs)) != world:
                raise SystemExit(f"ranks share a GPU under RCCL: {rccl_ranks}")
        wd.disarm()

    rccl_selftest = None
    if world == 1 and args.dist_selftest is not False:
        # RCCL executed on this box (one rank): communicator init on the device + the collectives the N > 1 path uses.  FIRST, on an
        # idle GPU and with torch's files already paged in by the import above (a fresh box takes a minute for the first import: that
        # is not RCCL's time), in a process of its own under a 60 s deadline.
        rccl_selftest = dist_selftest(float(os.environ.get("DPDF_BENCH_SELFTEST_CAP_S", "60")))
        mark("rccl_selftest_child")

    blob = synth_blob(backend.manifest(SR, NB), WEIGHT_SEED)
    model = backend.HipModel(SR, NB, blob, device=local_rank)
    if args.chunk:
        model.set_chunk_frames(args.chunk)
    if args.overlap >= 0:
        model.set_overlap(args.overlap)
    # the headline is the library's DEFAULT engine (GRU-64 throughput kernels on bf16 limbs since round 6), whatever the process environment says
    # (DPDF_GRU64_LIMBS changes the default of every handle: that is how the GPU suite is run under the other family); --fp32-mfma is the explicit A/B
    MODE = 0 if args.fp32_mfma else 3
    OTHER = 3 - MODE
    model.set_option("gru64_limbs", MODE)
    if args.no_fuse:
        model.set_fuse_dprnn(False)
    for kv in args.opt:
        k, v = kv.split("=")
        model.set_option(k, int(v))
    B, N = args.clips, int(CLIP_SECONDS * SR)
    T = model.num_frames(N)
    lo, hi = shard_range(B * world, world, rank)          # contiguous block of clips per rank
    wav_host = synth_clips(B, N, SR, WEIGHT_SEED + lo)
    wav = torch.from_numpy(wav_host).cuda()
    out = torch.empty_like(wav)
    gathered = None
    do_gather = world > 1 and not args.no_gather
    fallback = bool(args.fallback_reason)                 # this rank runs again on gloo because RCCL did not answer
    gather_note = "none (single GPU)" if world == 1 else ((("rccl" if args.backend == "nccl" else args.backend) + " gather to rank 0") if do_gather else "disabled")
    if fallback:
        gather_note = (f"FALLBACK gloo: {args.fallback_reason}; barriers / clocks over gloo, the enhanced PCM gathered to rank 0 over gloo through "
                       "pinned host staging ONCE behind the timed region (timed separately), not inside it")
    collective_error = None
    # the gather rides inside the timed region over RCCL (asynchronous, under the next step's compute); over the fallback's TCP
    # loopback it would be what is measured instead of the GPUs, so there it runs once, behind the region
    gather_in_timed = do_gather and not fallback

    # two output buffers: with N > 1 the RCCL gather of step i reads one while the engine writes step i+1 into the other
    outs = [out, torch.empty_like(out)] if gather_in_timed else [out, out]
    # The gather runs on RCCL's stream, the engine on its own private stream: nothing orders them but the host.  An event
    # recorded behind gather i is waited for (on the host; it is a whole step old by then) before step i+2 reuses its buffer.
    gather_done = [None, None]

    def step(i: int = 0) -> None:
        if gather_done[i & 1] is not None:
            gather_done[i & 1].synchronize()
            gather_done[i & 1] = None
        model.enhance_batch_device(wav.data_ptr(), B, N, outs[i & 1].data_ptr(), None)

    def sync() -> None:
        model.sync()
        torch.cuda.synchronize()

    mark("setup_model_and_clips")
    for _ in range(args.warmup):
        step()
    sync()
    mark("warmup_steps")
    if do_gather:
        if args.backend == "nccl":
            wd.arm(wd_s, "warm-up gather of the enhanced PCM over RCCL")
        try:
            gathered = gather_to_root(out, world, rank)
            torch.cuda.synchronize()
        except Exception as exc:
            # LOUD: the line still carries the compute figure (so a scaling run is not lost), but says so in two places
            do_gather = False
            collective_error = f"{type(exc).__name__}: {exc}"
            gather_note = f"FAILED, excluded from the timed region: {collective_error}"
            print(f"[bench.py] rank {rank}: the gather over {args.backend} FAILED ({collective_error}); timing compute only",
                  file=sys.stderr, flush=True)
        flags = [None] * world
        dist.all_gather_object(flags, bool(do_gather))
        do_gather = all(flags)                            # every rank takes the same path
        gather_in_timed = gather_in_timed and do_gather
        wd.disarm()

    # ---- the timed region: EXACTLY --steps steps, per-kernel profiling OFF ----
    rec0 = model.recovery_count
    if world > 1 and args.backend == "nccl":
        wd.arm(wd_s + 2.0 * args.steps, "timed region (barrier, steps, asynchronous gathers, barrier)")
    if world > 1:
        dist.barrier()
    sync()
    gather_ms = 0.0
    gather_events = []                 # (start, end) on torch's current stream around every timed gather: its device-side duration
    t0 = time.perf_counter()
    for i in range(args.steps):
        step(i)
        if gather_in_timed:
            model.sync()          # host waits for this rank's step i; the gather below is asynchronous (RCCL's stream),
            tg = time.perf_counter()
            ev0 = torch.cuda.Event(enable_timing=True); ev0.record()
            gathered = gather_to_root(outs[i & 1], world, rank, gathered)   # so it runs under the compute of step i+1
            ev = torch.cuda.Event(enable_timing=True); ev.record(); gather_done[i & 1] = ev
            gather_events.append((ev0, ev))
            gather_ms += 1e3 * (time.perf_counter() - tg)
    sync()
    if world > 1:
        dist.barrier()
    dt_local = time.perf_counter() - t0
    wd.disarm()
    recoveries = model.recovery_count - rec0          # calls of the timed region that were re-run after a device-side time-out (must be 0)
    mark("timed_region")
    dt = dt_local
    per_rank_ms = [1e3 * dt_local / args.steps]
    if world > 1:
        tmax = torch.tensor([dt], dtype=torch.float64, device="cuda" if args.backend == "nccl" else "cpu")
        dist.all_reduce(tmax, op=dist.ReduceOp.MAX)
        dt = float(tmax.item())
        allms = [None] * world
        gather_dev_ms = (sum(a.elapsed_time(b) for a, b in gather_events) / len(gather_events)) if gather_events else None
        dist.all_gather_object(allms, {"rank": rank, "ms_per_step": 1e3 * dt_local / args.steps, "gather_host_ms_per_step": gather_ms / args.steps,
                                       "gather_device_ms_per_step": gather_dev_ms})
        per_rank_ms = sorted(allms, key=lambda r: r["rank"])
    # the LAST timed step's output, copied out before anything else touches the buffers (parity block below)
    parity_slots = sorted({0, B // 2, B - 1})
    timed_out_host = {b: outs[(args.steps - 1) & 1][b].cpu().numpy() for b in parity_slots} if rank == 0 and args.steps > 0 else {}
    gather_check = None
    fallback_gather_ms = None
    if do_gather and fallback:
        tg = time.perf_counter()
        gathered = gather_to_root(outs[(args.steps - 1) & 1], world, rank, gathered)
        dist.barrier()
        fallback_gather_ms = 1e3 * (time.perf_counter() - tg)
    if do_gather:      # validate the gathered PCM once, outside the timed region: rank r's rows must be rank r's own output
        mine = torch.stack([outs[(args.steps - 1) & 1].double().sum(), outs[(args.steps - 1) & 1].double().abs().sum()]).cpu()
        sums = [None] * world
        dist.all_gather_object(sums, mine.tolist())
        if rank == 0:
            got = [[float(gathered[r].double().sum()), float(gathered[r].double().abs().sum())] for r in range(world)]
            gather_check = all(abs(a - b) <= 1e-9 * max(1.0, abs(b)) for g_, s_ in zip(got, sums) for a, b in zip(g_, s_))
            if not gather_check:
                print(f"[bench.py] gathered PCM does not match the ranks' outputs: {got} vs {sums}", file=sys.stderr, flush=True)

    # ---- per-kernel pass: the same pipelined steps again with HIP events around every launch class ----
    psteps = args.steps if args.profile_steps < 0 else args.profile_steps
    prof, prof_ms = {}, None
    if psteps > 0:
        model.profile(True)
        sync(); tp = time.perf_counter()
        for i in range(psteps):
            step(i)
        sync(); prof_ms = 1e3 * (time.perf_counter() - tp) / psteps
        prof = model.profile_report()
        model.profile(False)
    fused = not args.no_fuse
    # one extra serial step (not timed into `value`) to time the kernels without co-running streams
    iso_prof, iso_ms, kernel_stats_iso = None, None, None
    if rank == 0 and not args.no_isolated:
        model.set_overlap(0)
        model.profile(True)
        sync(); t1 = time.perf_counter(); step(); sync(); iso_ms = 1e3 * (time.perf_counter() - t1)
        iso_prof = model.profile_report()
        model.profile(False)
        model.set_overlap(args.overlap if args.overlap >= 0 else 27)
    # The OTHER GRU-64 kernel family beside the headline (never `value`): the same pipelined steps with dpdf_set_option gru64_limbs = OTHER
    # (0: the fp32-MFMA kernels of gru_scan.h, the default of rounds 1-5; 3: the bf16-limb kernels of gru_limb.h) -- its own timing, its own
    # per-kernel pass, its own parity block
    limb = None
    if rank == 0 and not args.no_isolated and not args.no_fuse:
        model.set_option("gru64_limbs", OTHER)
        step(); sync()
        nl = max(1, min(args.steps, 3))
        t1 = time.perf_counter()
        for i in range(nl):
            step(i)
        sync(); ms_l = 1e3 * (time.perf_counter() - t1) / nl
        limb_out = {b: outs[(nl - 1) & 1][b].cpu().numpy() for b in sorted({0, B // 2, B - 1})}
        model.profile(True)
        step(); sync()
        limb_prof = model.profile_report()
        model.profile(False)
        model.set_overlap(0); model.profile(True)
        step(); sync()
        limb_iso = model.profile_report()
        model.profile(False); model.set_overlap(args.overlap if args.overlap >= 0 else 27)
        model.set_option("gru64_limbs", MODE)
        limb = {"ms_per_step": ms_l, "value": B * T / (ms_l * 1e-3), "out": limb_out, "prof": limb_prof, "iso": limb_iso}

    mark("per_kernel_event_passes")
    # ---- SURVEY 8(d)'s full metric: the same steps INCLUDING H2D of the noisy PCM and D2H of the enhanced PCM ----
    # Through the PRODUCT: the library's own host-pointer call (dpdf_enhance_batch: numpy block in, numpy block out, pageable
    # memory), which pipelines upload / compute / download over time slices inside the library (pinned staging ring, copy
    # threads, per-chunk STFT / iSTFT: csrc/dpdf_model.hip enhance_impl).  Nothing is staged or overlapped by this file.
    pcie = None
    if world == 1 and not args.no_pcie:
        def run_host(nsteps: int):
            sync(); t_ = time.perf_counter()
            y = None
            for _ in range(nsteps):
                y = model.enhance_batch(wav_host)
            return time.perf_counter() - t_, y

        run_host(1)
        dtp, y_host = run_host(args.steps)
        model.set_option("host_pipe", 0)
        run_host(1)
        dtp0, _ = run_host(max(1, min(args.steps, 3)))
        model.set_option("host_pipe", 1)
        dtp0 /= max(1, min(args.steps, 3))
        ref_slots = {b: timed_out_host[b] for b in timed_out_host} if timed_out_host else {}
        pcie = {"value_incl_pcie": B * T * args.steps / dtp, "ms_per_step_incl_pcie": 1e3 * dtp / args.steps,
                "note": "dpdf_enhance_batch with HOST pointers (pageable numpy block in and out), every step: the library pipelines "
                        "H2D / compute / D2H over time slices itself; includes the exposed first upload and last download",
                "bytes_per_step_each_way": int(B * N * 4),
                "ms_per_step_unpipelined": 1e3 * dtp0,
                "unpipelined_note": "the same call with dpdf_set_option host_pipe=0: one pageable upload, compute, one pageable download",
                "finite_output": bool(np.isfinite(y_host).all()),
                "max_abs_diff_vs_hbm_resident_output": (max(float(np.abs(y_host[b] - ref_slots[b]).max()) for b in ref_slots) if ref_slots else None)}

    mark("pcie_inclusive_passes")
    if rank == 0:
        finite = bool(torch.isfinite(out).all().item())
        total_frames = world * B * T * args.steps
        value = total_frames / dt
        # Dominant kernel family: the GRU-64 scans of the DPRNN blocks (reference layers.py:159-196).  With the
        # fused epilogues they are three kernels; rocprofv3 --kernel-trace reports the same three names:
        #   gru64_scan_kernel      intra-band forward direction            49 152 FLOP per (row, step)
        #   gru64_epi_kernel<2>    intra-band backward + fc_intra + LN     49 152 + 2*64*128 FLOP
        #   gru64_epi_kernel<1>    inter-band + fc_inter + LN              49 152 + 2*64*64 FLOP
        # rows*steps per step of the bench: NB blocks x B*T frames x (48 DF + 8 ERB) band positions.
        rs = NB * (B * T) * (48 + 8)
        # Round 5 (opt-in then, the default since round 6): the same three launches on bf16 LIMBS (gru_limb.h, option gru64_limbs): every fp32 product is formed from
        # 3 x 3 bf16 limbs, six v_mfma_f32_16x16x32_bf16 per term, fp32 accumulation -- same algorithmic (fp32) FLOPs, six times as
        # many matrix FLOPs issued, on a pipe with 16 x the fp32 rate.  `flop` below is the ALGORITHMIC fp32 count per (row, step);
        # `issued` = flop x 6 is what the bf16 pipe executes and what the roofline prices against the bf16 peak.
        #   gru64_l3_kernel<0>     intra-band forward + its half of fc_intra        49 152 + 2*64*64
        #   gru64_l3_kernel<2>     intra-band backward + its half of fc_intra + LN  49 152 + 2*64*64
        #   gru64_l3_kernel<1>     inter-band + fc_inter + LN                       49 152 + 2*64*64
        fam = {
            "gru64_scan_kernel": GRU64_FLOP_PER_ROW_STEP * (1 if fused else 3),
            "gru64_epi_kernel<2>": GRU64_FLOP_PER_ROW_STEP + 2 * 64 * 128,
            "gru64_epi_kernel<1>": GRU64_FLOP_PER_ROW_STEP + 2 * 64 * 64,
            "gru64_scan_gi_kernel": GRU64_FLOP_PER_ROW_STEP,      # small --clips only: hoisted input GEMM + h-part scan
            "gru64_l3_kernel<0>": GRU64_FLOP_PER_ROW_STEP + 2 * 64 * 64,
            "gru64_l3_kernel<2>": GRU64_FLOP_PER_ROW_STEP + 2 * 64 * 64,
            "gru64_l3_kernel<1>": GRU64_FLOP_PER_ROW_STEP + 2 * 64 * 64,
        }
        is_limb = lambda k: k.startswith("gru64_l3_kernel")

        def kernel_stats(p, nsteps):
            out_ = {}
            for kname, flop_rs in fam.items():
                sel = {k: v for k, v in p.items() if k.split("/")[0] == kname}
                ms_ = sum(v[0] for v in sel.values()); n_ = sum(v[1] for v in sel.values())
                if n_:
                    fl = flop_rs * rs * nsteps
                    mult = LIMB_TERMS if is_limb(kname) else 1
                    out_[kname] = {"ms_total": ms_, "launches": n_, "avg_launch_ms": ms_ / n_,
                                   "flop_per_launch": fl / n_, "tflops": fl / (ms_ * 1e-3) / 1e12,
                                   "issued_flop_per_launch": mult * fl / n_, "issued_tflops": mult * fl / (ms_ * 1e-3) / 1e12,
                                   "peak": BF16_MFMA_PEAK_TFLOPS if is_limb(kname) else FP32_MFMA_PEAK_TFLOPS}
            return out_

        line = {
            "metric": METRIC, "value": value, "unit": "frames/s", "n_gpus": world, "steps": args.steps,
            "warmup": args.warmup, "ms_per_step": 1e3 * dt / args.steps, "higher_is_better": True,
            "scaling": "weak", "vs_baseline": None, "dtype": "f32", "data": "synthetic",
            "config": {"workload": f"{MODEL} @16 kHz, {B} clips x {CLIP_SECONDS:g} s per GPU (T={T} frames/clip), "
                                   "seeded synthetic weights + clips, inputs/outputs resident in HBM",
                       "clips_per_gpu": B, "frames_per_clip": T, "chunk_frames": args.chunk,
                       "sharding": f"utterances, contiguous blocks per rank; collective: {gather_note}"},
            "finite_output": finite,
        }
        # `value` is the contract's figure: inputs and outputs resident in HBM when the timed region starts.  SURVEY 8(d)
        # words the metric with the H2D / D2H of the PCM inside: that figure is `value_incl_pcie` (measured below in the
        # same run); `value_hbm_resident` repeats `value` under an explicit name.
        line["value_hbm_resident"] = value
        if MODE == 3:
            # every value, state and accumulator of the path is fp32 (the analysis DFT float64); the PRODUCTS of the GRU-64 throughput kernels are formed
            # from three bf16 limbs per operand -- exact where the fp32 MFMA rounds (float64_recurrence_error below: not narrower than fp32)
            line["dtype"] = "f32 (GRU-64 products as bf16x3 limbs, fp32 accumulate)"
            line["float64_recurrence_error"] = float64_recurrence_error()
        else:
            line["ab_mode"] = "--fp32-mfma: THIS RUN times the fp32-MFMA GRU-64 kernels (dpdf_set_option gru64_limbs = 0), not the default engine"
        if not args.no_parity and timed_out_host:
            line["parity"] = parity_vs_oracle(blob, wav_host, timed_out_host, parity_slots, WEIGHT_SEED + lo)
            mark("parity_vs_oracle")
            if not line["parity"]["ok"]:
                print(f"[bench.py] PARITY FAILURE on the timed shape: {line['parity']}", file=sys.stderr, flush=True)
        if pcie is not None:
            line.update({"value_incl_pcie": pcie["value_incl_pcie"], "ms_per_step_incl_pcie": pcie["ms_per_step_incl_pcie"]})
            line["pcie"] = pcie
        if world > 1:
            line["multi_gpu"] = {"backend": "rccl" if args.backend == "nccl" else (args.backend + (" (FALLBACK: RCCL did not answer)" if fallback else "")),
                                 "fallback_reason": args.fallback_reason or None, "fallback_gather_ms_once_outside_timed_region": fallback_gather_ms,
                                 "gather_inside_timed_region": bool(gather_in_timed), "rccl_ranks": rccl_ranks,
                                 "per_rank": per_rank_ms, **multi_gpu_summary(per_rank_ms), "collective_ok": bool(do_gather) if not args.no_gather else None,
                                 "collective_error": collective_error, "gathered_matches_rank_outputs": gather_check,
                                 "gathered_shape": list(gathered.shape) if gathered is not None else None}
        ks = kernel_stats(prof, psteps) if prof else {}
        dom = next((k for k in ("gru64_l3_kernel<2>", "gru64_epi_kernel<2>", "gru64_scan_kernel", "gru64_scan_gi_kernel") if k in ks), None)
        if dom is not None:
            if iso_prof is not None:
                kernel_stats_iso = kernel_stats(iso_prof, 1)
            ms, calls = ks[dom]["ms_total"], ks[dom]["launches"]
            achieved = ks[dom]["issued_tflops"]
            peak = ks[dom]["peak"]
            fam_ms = sum(v["ms_total"] for v in ks.values())
            fam_flop = sum(v["flop_per_launch"] * v["launches"] for v in ks.values())
            # HBM bytes per launch from the committed rocprofv3 PMC passes (FETCH_SIZE / WRITE_SIZE collected in
            # separate --pmc runs of this same command, gfx950 x2 read correction applied; profiles/README.md)
            traffic, traffic_note = None, "no PMC summary in profiles/ for this kernel"
            try:
                pmc_all = json.loads((ROOT / "profiles" / "pmc_summary.json").read_text())
                pmc = next(v for k, v in pmc_all.items() if k.replace("void ", "") == dom)
                traffic = pmc["hbm_bytes_per_dispatch_corrected"]
                traffic_note = "bytes/launch, profiles/pmc_summary.json (offline rocprofv3 --pmc FETCH_SIZE / WRITE_SIZE passes)"
            except Exception:
                pass
            # algorithmic bytes: x row in, (hf row in,) y row out = 256 B each per (row, step)
            alg_bytes = {"gru64_scan_kernel": 2 * 256, "gru64_epi_kernel<2>": 3 * 256, "gru64_epi_kernel<1>": 2 * 256,
                         "gru64_scan_gi_kernel": 256 + 768 + 256, "gru64_l3_kernel<2>": 3 * 256}[dom]
            serial_mode = args.overlap == 0
            roofline = {
                "bound": "mfma", "kernel": dom + " (all launches, DF + ERB branch)",
                "achieved": achieved, "peak": peak, "unit": "TFLOP/s",
                "frac": achieved / peak, "traffic": traffic, "traffic_note": traffic_note,
                "accounting": (f"limb kernel: achieved = {LIMB_TERMS} x the algorithmic fp32 FLOPs per launch (the bf16 MFMAs actually issued) / launch duration, "
                               f"against the dense bf16 MFMA peak {BF16_MFMA_PEAK_TFLOPS:g}; `useful_fp32_tflops` is the algorithmic rate, which the fp32 pipe "
                               f"({FP32_MFMA_PEAK_TFLOPS} peak) could not reach" if is_limb(dom) else "fp32 MFMA kernel against the fp32 MFMA peak"),
                "useful_fp32_tflops": ks[dom]["tflops"],
                "algorithmic_bytes_per_launch": alg_bytes * rs * psteps / calls,
                "avg_launch_ms": ms / calls, "launches": calls, "flop_per_launch": ks[dom]["flop_per_launch"],
                "timing": f"HIP events on the launching stream around every launch of {psteps} steps run right after the timed "
                          "region in the same execution shape (the timed region itself runs with these events off: "
                          f"{1e3 * dt / args.steps:.2f} ms/step timed vs {prof_ms:.2f} ms/step with events)",
                "reproduce": (banked_trace(("fp32mfma_" if MODE == 0 else "") + "serial") if serial_mode else banked_trace(("fp32mfma_" if MODE == 0 else "") + "pipelined"))
                             + ": rocprofv3 --kernel-trace --stats of `python bench.py --no-isolated --no-other-configs --no-cpu-baseline "
                               "--no-pcie" + (" --fp32-mfma" if MODE == 0 else "") + (" --overlap 0`" if serial_mode else "`") + " -- every launch of that run has this execution "
                               "shape, so the CSV's AverageNs for the kernel is this avg_launch_ms (profiles/README.md)",
                "gru64_family": {k: {"avg_launch_ms": round(v["avg_launch_ms"], 4), "launches": v["launches"],
                                     "useful_fp32_tflops": round(v["tflops"], 1), "issued_tflops": round(v["issued_tflops"], 1),
                                     "frac_of_its_pipe_peak": round(v["issued_tflops"] / v["peak"], 3)} for k, v in ks.items()},
                "gru64_family_tflops": fam_flop / (fam_ms * 1e-3) / 1e12 if fam_ms else None,
                "whole_path_fp32_equiv_tflops": value * FLOP_PER_FRAME / 1e12 / world,
                "whole_path_over_fp32_peak": value * FLOP_PER_FRAME / 1e12 / FP32_MFMA_PEAK_TFLOPS / world,
                "whole_path_note": "frames/s x algorithmic fp32 FLOP per frame (SURVEY 8(d)) over the fp32 MFMA peak -- north_star's yardstick; with the "
                                   "GRU-64 products on the bf16 pipe it is no longer an upper bound of 1",
                # the three GRU-64 kernels' algorithmic FLOPs over the WALL time of a step: a lower bound on what
                # they achieve while sharing the chip (unlike per-launch durations it only goes up when throughput goes up)
                "gru64_family_wallclock_over_fp32_peak": fam_flop / psteps / (dt / args.steps) / 1e12 / FP32_MFMA_PEAK_TFLOPS,
                "per_class_ms_per_step": {k: round(v[0] / psteps, 3) for k, v in sorted(prof.items())},
            }
            if kernel_stats_iso is not None:
                ki = kernel_stats_iso
                roofline["frac_isolated"] = round(ki[dom]["issued_tflops"] / ki[dom]["peak"], 4) if dom in ki else None
                roofline["frac_note"] = ("`frac` divides by the launch duration seen INSIDE the 4-stream pipeline, where the kernel "
                                         "shares the CUs with three other streams (faster pipeline => longer individual launches); "
                                         "`frac_isolated` is the same kernel, same launches, run back to back in the extra serial "
                                         f"step (= {banked_trace('serial')}, the --overlap 0 run); `whole_path_over_fp32_peak` is "
                                         "frames/s x FLOP/frame over the fp32 MFMA peak")
                roofline["roofline_isolated"] = {
                    "note": "one extra step AFTER the timed region with the stream pipeline switched off (kernels back to back)",
                    "ms_per_step": iso_ms,
                    "kernels": {k: {"avg_launch_ms": round(v["avg_launch_ms"], 4), "useful_fp32_tflops": round(v["tflops"], 1),
                                    "issued_tflops": round(v["issued_tflops"], 1), "frac": round(v["issued_tflops"] / v["peak"], 3)} for k, v in ki.items()},
                    "per_class_ms_per_step": {k: round(v[0], 3) for k, v in sorted(iso_prof.items())},
                }
            line["roofline"] = roofline
            if limb is not None:
                lk, li = kernel_stats(limb["prof"], 1), kernel_stats(limb["iso"], 1)
                ld = "gru64_l3_kernel<2>" if OTHER == 3 else "gru64_epi_kernel<2>"
                lpeak = BF16_MFMA_PEAK_TFLOPS if OTHER == 3 else FP32_MFMA_PEAK_TFLOPS
                lpar = parity_vs_oracle(blob, wav_host, limb["out"], sorted(limb["out"]), WEIGHT_SEED + lo) if (not args.no_parity and timed_out_host) else None
                what3 = ("the three GRU-64 throughput launches of a DPRNN block form every fp32 product from three bf16 limbs per operand (v = hi + mid + lo exactly; six "
                         "v_mfma_f32_16x16x32_bf16 per term, fp32 accumulate): gru_limb.h -- fp32-exact products, closer to a float64 recurrence than the fp32-MFMA kernels "
                         "(float64_recurrence_error)")
                what0 = ("the GRU-64 throughput launches as v_mfma_f32_16x16x4_f32 kernels (gru_scan.h): the default engine of rounds 1-5, kept as a mode "
                         "(dpdf_set_option gru64_limbs 0 / DPDF_GRU64_LIMBS=0) and measured here so that both families are on one line")
                line["limb_kernels" if OTHER == 3 else "fp32_mfma_kernels"] = {
                    "what": f"NOT the headline: the same step with dpdf_set_option(gru64_limbs, {OTHER}) -- " + (what3 if OTHER == 3 else what0),
                    "value": limb["value"], "ms_per_step": limb["ms_per_step"],
                    "headline_over_this": (limb["ms_per_step"] * 1e-3) / (dt / args.steps),
                    "dtype": "f32 (bf16x3 limbs, fp32 accumulate)" if OTHER == 3 else "f32",
                    "parity": lpar,
                    "float64_recurrence_error": line.get("float64_recurrence_error") or float64_recurrence_error(),
                    "roofline": None if ld not in lk else {
                        "bound": "mfma", "kernel": ld, "achieved": lk[ld]["issued_tflops"], "peak": lpeak, "unit": "TFLOP/s",
                        "frac": lk[ld]["issued_tflops"] / lpeak,
                        "frac_isolated": (li[ld]["issued_tflops"] / lpeak) if ld in li else None,
                        "useful_fp32_tflops": lk[ld]["tflops"], "useful_fp32_tflops_isolated": li[ld]["tflops"] if ld in li else None,
                        "avg_launch_ms": lk[ld]["avg_launch_ms"], "launches": lk[ld]["launches"],
                        "accounting": (f"achieved = {LIMB_TERMS} x the algorithmic fp32 FLOPs per launch (the bf16 MFMAs issued) / launch duration, against the dense bf16 peak"
                                       if OTHER == 3 else "algorithmic fp32 FLOPs per launch / launch duration, against the fp32 MFMA peak"),
                        "family": {k: {"avg_launch_ms": round(v["avg_launch_ms"], 4), "avg_launch_ms_isolated": round(li[k]["avg_launch_ms"], 4) if k in li else None,
                                       "useful_fp32_tflops": round(v["tflops"], 1), "issued_tflops": round(v["issued_tflops"], 1)} for k, v in lk.items()}},
                }
                if lpar is not None and not lpar["ok"]:
                    print(f"[bench.py] PARITY FAILURE of the gru64_limbs = {OTHER} kernels: {lpar}", file=sys.stderr, flush=True)
        else:
            line["roofline"] = None
            print("[bench.py] no GRU-64 kernel launches were profiled (--profile-steps 0?): the roofline block is empty", file=sys.stderr)
        if world == 1 and not args.no_cpu_baseline:
            line["cpu_baseline"] = cpu_baseline(blob, args.cpu_clip_seconds, args.cpu_clips_per_thread)
            mark("cpu_baseline")
            # the reference's own CPU runtime, if this box has it (it does not offline: then the leg is reported as absent, not faked)
            onnx_path = os.environ.get("DPDFNET_ONNX", "")
            try:
                if not onnx_path or not Path(onnx_path).is_file():
                    raise FileNotFoundError("DPDFNET_ONNX not set or not a file")
                line["cpu_baseline"]["reference_runtime"] = ort_baseline(onnx_path)
            except Exception as exc:
                line["cpu_baseline"]["reference_runtime"] = {"kind": "ort", "available": False,
                                                              "why": f"{type(exc).__name__}: {exc}"[:200]}
        if rccl_selftest is not None:
            line["rccl_selftest"] = rccl_selftest
            line["rccl_init_ok"] = bool(rccl_selftest.get("rccl_init_ok"))
        if world == 1 and not args.no_pcie:
            model.close()       # the public API builds its own (cached) handle: give it the device
            try:
                line["public_api"] = public_api_pass(B, max(1, args.steps), timed_out_host)
                line["value_public_api"] = line["public_api"]["value_public_api"]
                line["public_api_over_hbm_resident"] = line["value_public_api"] / value
            except Exception as exc:
                line["public_api"] = {"error": f"{type(exc).__name__}: {exc}"}
            mark("public_api_child")
        if world == 1 and not args.no_other_configs and not args.no_isolated:
            model.close()       # the side configurations get the device to themselves (the headline engine's 33 GB workspace and four streams go first)
            try:
                line["other_configs"] = other_configs()
            except Exception as exc:  # never lose the headline line over the side measurements
                line["other_configs"] = {"error": f"{type(exc).__name__}: {exc}"}
            mark("other_configs_children")
        # forward-progress hygiene: a GRU-256 cluster exchange / hop hand-off that timed out costs ~1 s and a re-run on the non-spinning
        # kernels (dpdf_recovery_count).  In the timed region that would silently be a wrong measurement: it is on the line, and fatal.
        line["recovery_count"] = recoveries
        timeline["total"] = round(time.perf_counter() - _PROC_T0, 2)
        line["timeline_s"] = timeline
        print(json.dumps(line), flush=True)
        if recoveries:
            print(f"[bench.py] FATAL: {recoveries} call(s) inside the timed region were re-run after a device-side time-out "
                  "(dpdf_recovery_count): `value` includes the time-out and the re-run and is not a measurement", file=sys.stderr, flush=True)
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()
    model.close()
    if rank == 0 and recoveries:
        raise SystemExit(3)


if __name__ == "__main__":
    main()
