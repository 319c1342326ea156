#!/usr/bin/env python3
"""Headline benchmark: masked utterances / second through the inpainting hot path on MI355X.

One "step" = one pass of the hot path over one batch of synthetic GRID-shaped input that is
already resident in HBM: fused STFT / log-spectrum front end -> 3 x BLSTM-250 forward
(hoisted fp32-MFMA input GEMMs + recurrent kernel) -> 500->257 projection + sequence mask ->
L1 loss (what the reference's `infer` fetches per batch, inference.py:131, minus the
waveform reconstruction).  Workload = BASELINE.json configs[1]: audio-only 3xBLSTM-250
inpainter on 3 s / 16 kHz clips with one 400 ms gap each.

  python bench.py [--gpus N] [--steps K] [--warmup W] [--batch B]

For N > 1 launch with torch.distributed.run (one rank per GPU); utterances are sharded across
ranks with no data-path collective (weak scaling: per-GPU batch fixed).  Rank 0 prints ONE JSON
line.  Its `also` block reports the sizes the reference and BASELINE.json name (inference at 100 and
32 utterances, AV training at 32 utterances per GPU -- with the gradient all-reduce when N > 1) and two
mid sizes (inference at 128 and 1024 utterances), plus the LWS phase reconstruction of 32 enhanced utterances (the step
after the path in the reference's default `infer`), each
with its own ms_per_step, measured after the headline.  `roofline` is measured live with HIP events on the launch stream around the dominant
kernel; `cpu_baseline` times the CPU oracle (a numpy port of the reference graph) on a bounded
sample of the same workload on this node's host cores.
"""
import argparse
import json
import os
import sys
import time

import numpy as np

ROOT = os.path.dirname(os.path.abspath(__file__))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

N_SAMPLES = 48000          # 3 s @ 16 kHz
T_FRAMES = 250
F_BINS = 257
GAP_FRAMES = 33            # 400 ms (dataset_generator.py:16-17,73)
H = 250
FP32_MFMA_PEAK_TFLOPS = 157.3   # MI355X_MICROARCH.md: v_mfma_f32_32x32x2_f32, dense
HBM_PEAK_GBS = 8000.0


def device_copy_rate(torch, device, mib=4096, reps=5, kernel="float4"):
    """Read + write bytes per second of a streaming copy of `mib` MiB: what a pure streaming kernel reaches on this GPU,
    the practical ceiling for the HBM-bound kernels next to the 8 TB/s of the data sheet.  kernel = "float4": the C ABI's
    avsi_diag_copy_f32 (16 bytes per lane, four accesses in flight, a grid sized to the chip -- the shape
    MI355X_MICROARCH.md quotes 6.29 TB/s for); "torch": torch's own copy kernel (round 3's yardstick, ~20 % lower)."""
    from avsi_amd import _lib
    src = torch.empty(mib << 18, dtype=torch.float32, device=device).normal_()
    dst = torch.empty_like(src)

    def copy():
        if kernel == "torch":
            dst.copy_(src)
        else:
            _lib.check(_lib.lib().avsi_diag_copy_f32(_lib.ptr(src), _lib.ptr(dst), src.numel(), _lib.stream_ptr()),
                       "avsi_diag_copy_f32")
    copy()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(reps):
        copy()
    e1.record()
    torch.cuda.synchronize(device)
    return 2.0 * src.numel() * 4 * reps / (e0.elapsed_time(e1) * 1e-3) / 1e9


def algorithmic_flops(batch, input_dim=257):
    """forward FLOPs of the gate GEMMs, split by kernel, per `batch` utterances."""
    d = [input_dim, 2 * H, 2 * H]
    gemm_in = [2.0 * d[l] * (4 * H) * 2 * T_FRAMES * batch for l in range(3)]       # x_t . Wx, both dirs
    rec = 2.0 * H * (4 * H) * 2 * T_FRAMES * batch                                   # h_{t-1} . Wh, per layer
    proj = 2.0 * (2 * H) * F_BINS * T_FRAMES * batch
    return gemm_in, rec, proj


class KernelTimer:
    """HIP-event pairs on the launch stream (torch's current stream is the stream the C ABI
    launches on), grouped by kernel name.  Events come from a pool that reset() fills OUTSIDE the timed
    region: creating a few thousand events inside it (70 launches per U-Net step) stalls the host for ~50 ms
    once the runtime has to grow its event pool."""

    def __init__(self, torch):
        self.torch = torch
        self.events = {}
        self.pool = []

    def _event(self):
        return self.pool.pop() if self.pool else self.torch.cuda.Event(enable_timing=True)

    def wrap(self, name, fn):
        def timed(*a, **kw):
            s, e = self._event(), self._event()
            s.record()
            out = fn(*a, **kw)
            e.record()
            self.events.setdefault(name, []).append((s, e))
            return out
        return timed

    def reset(self, steps, warmup):
        """After the warm-up: recycle its events and create what `steps` timed steps will need on top."""
        used = sum(len(v) for v in self.events.values())
        for v in self.events.values():
            for s, e in v:
                self.pool += [s, e]
        self.events.clear()
        need = 2 * (used // max(warmup, 1) + 8) * steps
        while len(self.pool) < need:
            self.pool.append(self.torch.cuda.Event(enable_timing=True))

    def totals(self):
        return {k: (sum(s.elapsed_time(e) for s, e in v), len(v)) for k, v in self.events.items()}


def synth_batch(torch, batch, seed, device):
    """Seeded synthetic GRID-shaped inputs generated on the device."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    wav = torch.clamp(torch.round(torch.randn(batch, N_SAMPLES, generator=g, device=device) * 3000.0),
                      -32768, 32767)
    masks = torch.ones(batch, T_FRAMES, F_BINS, device=device)
    starts = torch.randint(0, T_FRAMES - GAP_FRAMES, (batch,), generator=g, device=device)
    t = torch.arange(T_FRAMES, device=device)[None, :]
    gap = (t >= starts[:, None]) & (t < starts[:, None] + GAP_FRAMES)
    masks[gap] = 0.0
    return wav, masks


def cpu_baseline(torch, model, wav, masks, mean, std, sample, pred_gpu):
    """Time the CPU oracle (float32 numpy, explicit per-step loop = the reference's
    stack_bidirectional_dynamic_rnn schedule) on `sample` utterances of the same workload, in batches of 32
    (scripts/inference.sh:7) and of 8 (scripts/config/blstm.config:8), and use its output as the checker for
    `pred_gpu`: the first `sample` rows of the prediction of the LAST TIMED step (so the kernels that are
    checked are the kernels that were timed)."""
    from oracle import blstm as OB
    from oracle import frontend as OF
    params = model.layout.unflatten_to_oracle_params(model.variables.flat.cpu().numpy())
    w = wav[:sample].cpu().numpy()
    m = masks[:sample].cpu().numpy()
    mean_h, std_h = mean.cpu().numpy(), std.cpu().numpy()
    OB.model_forward(w[:8], m[:8], mean_h, std_h, np.full(8, T_FRAMES), params, dtype=np.float32)   # warm-up

    def run(n, cpu_batch):
        preds = []
        t0 = time.perf_counter()
        for i in range(0, n, cpu_batch):
            out = OB.model_forward(w[i:i + cpu_batch], m[i:i + cpu_batch], mean_h, std_h,
                                   np.full(len(w[i:i + cpu_batch]), T_FRAMES), params, dtype=np.float32)
            preds.append(out['prediction'])
        return np.concatenate(preds), time.perf_counter() - t0

    pred32, dt32 = run(sample, 32)
    n8 = max(8, (sample // 3) // 8 * 8)
    _, dt8 = run(n8, 8)
    pred_cpu = pred32.astype(np.float64)
    lm_cpu = OF.logmel_of_prediction(pred_cpu, mean_h, std_h)
    lm_gpu = OF.logmel_of_prediction(pred_gpu.astype(np.float64), mean_h, std_h)
    rms = float(np.sqrt(np.mean((lm_cpu - lm_gpu) ** 2)))
    try:
        cores = len(os.sched_getaffinity(0))
    except AttributeError:
        cores = os.cpu_count()
    # best-case CPU line: the same network shape through torch's fused CPU LSTM (oneDNN), random
    # weights, network only (no front end) -- an upper bound for what a CPU port could reach.  Threads pinned to
    # the physical share of this process (an unpinned run on a 128-thread host was SLOWER than the numpy loop:
    # oversubscription), whole sample as one batch per call.
    fused = None
    try:
        threads_before = torch.get_num_threads()
        torch.set_num_threads(max(1, min(cores, 32)))
        with torch.no_grad():
            F = model.audio_feat_dim
            net = torch.nn.LSTM(F, 250, num_layers=3, bidirectional=True, batch_first=True)
            proj = torch.nn.Linear(500, F)
            x = torch.randn(sample, T_FRAMES, F)
            best = None
            for fb in (32, 128):
                proj(net(x[:fb])[0])
                t1 = time.perf_counter()
                for i in range(0, sample, fb):
                    proj(net(x[i:i + fb])[0])
                rate = sample / (time.perf_counter() - t1)
                if best is None or rate > best[0]:
                    best = (rate, fb)
            fused = {"value": best[0], "unit": "utterances/s", "threads": torch.get_num_threads(),
                     "what": "torch.nn.LSTM + Linear forward, float32, batches of %d (best of 32 / 128)" % best[1]}
    except Exception as e:   # a reported extra, never a reason to lose the bench line
        fused = {"error": str(e)[:200]}
    # The rest of this process only launches GPU work.  Back at the default thread count, every small host-side
    # tensor op of a training step woke the whole OpenMP pool on a box that grants this process 16 cores, and the
    # pool's spin-waiting starved the launching thread (training at 32 utterances: 8.1 instead of 7.4 ms per step).
    torch.set_num_threads(1)
    return {"value": sample / dt32, "unit": "utterances/s", "cores": cores, "kind": "port",
            "sample": "%d utterances in batches of 32, float32 numpy oracle (per-step loop), %.1f s" % (sample, dt32),
            "batch_8": {"value": n8 / dt8, "unit": "utterances/s",
                        "sample": "%d utterances in batches of 8, %.1f s" % (n8, dt8)},
            "best_case_fused_cpu": fused}, rms


def bench_unet(args, torch, dist, rank, world, device):
    """U-Net spectrogram inpainter (UNetFConvModel), inference, mixed 100-1600 ms gap masks."""
    import avsi_amd  # noqa: F401
    from avsi_amd import models, ops
    from avsi_amd import audio_processing as ap_mod
    B = args.batch
    model, step = unet_setup(torch, models, ap_mod, B, 4321 + rank, device)
    timer = KernelTimer(torch)
    if B >= 256:      # below that a step is launch-bound and the per-call events would dominate what they measure
        # the matrix-core convolutions only (11 of ~70 launches, 70 % of the kernel time): events around every launch of
        # the step cost 0.4 of its 4.4 ms (AVSI_BENCH_UNET_ALL=1 times them all, for the per-kernel table of DESIGN 4.5)
        names = ("conv2d", "conv2d_thin_mfma")
        if os.environ.get("AVSI_BENCH_UNET_ALL", "0") == "1":
            names += ("conv2d_thin", "conv2d_thin_relu_pool", "colstats", "bn_act", "bn_act_pool", "maxpool2")
        for name in names:
            setattr(ops, name, timer.wrap(name, getattr(ops, name)))

    for _ in range(args.warmup):
        step()
    timer.reset(args.steps, args.warmup)
    if world > 1:
        dist.barrier()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(args.steps):
        loss = step()
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    elapsed = time.perf_counter() - t0
    if world > 1:
        tmax = torch.tensor([elapsed], device=device if dist.get_backend() == "nccl" else "cpu", dtype=torch.float64)
        dist.all_reduce(tmax, op=dist.ReduceOp.MAX)
        elapsed = float(tmax.item())
    if rank == 0:
        totals = timer.totals()
        flops = UNET_FLOPS_PER_CLIP * B * args.steps
        print(json.dumps({
            "metric": "spectrogram clips/sec (U-Net inference: front end + 13 conv layers + L1 loss)",
            "value": B * world * args.steps / elapsed, "unit": "clips/s", "n_gpus": world, "steps": args.steps,
            "warmup": args.warmup, "ms_per_step": elapsed / args.steps * 1e3, "higher_is_better": True, "scaling": "weak",
            "vs_baseline": None, "dtype": "f32", "data": "synthetic",
            "config": {"workload": "configs[4]: U-Net (fconv) spectrogram inpainter, 1.024 s 16 kHz clips, 128 x 128 log-spectrogram, "
                                   "one 100-800 ms gap", "per_gpu_batch": B, "global_batch": B * world,
                       "parallelism": "dp%d" % world},
            "loss_func": float(loss), "algorithmic_TFLOP/s": flops / elapsed / 1e12,
            "kernel_ms_per_step": {k: v[0] / args.steps for k, v in totals.items()}}))
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()


def profiled_traffic(kernel_key, batch):
    """(HBM bytes per launch, provenance) from the committed PMC passes (profiles/r*_traffic_b<batch>.json:
    FETCH_SIZE and WRITE_SIZE collected in separate rocprofv3 --pmc runs of this same command, gfx950 correction
    applied there; counters cannot be read from inside the process that is being timed).  The provenance names
    the file and the git commit the profile was taken at, so a stale figure is visible as such.  (None, None)
    when no profile exists for this batch size."""
    import glob
    files = sorted(glob.glob(os.path.join(ROOT, "profiles", "r*_traffic_b%d.json" % batch)))
    if not files:
        return None, None
    try:
        prof = json.load(open(files[-1]))
        for name, v in prof["kernels"].items():
            if name in kernel_key or kernel_key in name:
                return v["hbm_bytes_per_launch_avg"], {"file": "profiles/" + os.path.basename(files[-1]),
                                                       "commit": prof.get("commit"), "collected": prof.get("collected")}
    except Exception:
        return None, None
    return None, None


def time_steps(torch, step, steps, warmup):
    """ms per step of `step()` on the current device (single rank: the named-workload entries of `also`)."""
    for _ in range(warmup):
        step()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        step()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) / steps * 1e3


def _all_reduce(torch, dist, t, op):
    """In-place all-reduce of a device tensor: on the device over RCCL, staged through the host under gloo (the
    single-GPU rehearsal of the multi-rank path, tests/test_bench_contract_gpu.py)."""
    if dist.get_backend() == "nccl":
        dist.all_reduce(t, op=op)
    else:
        h = t.cpu()
        dist.all_reduce(h, op=op)
        t.copy_(h)
    return t


def time_steps_all_ranks(torch, dist, world, step, steps, warmup):
    """ms per step the way the driver contract times the headline: barrier + synchronize on both sides, MAX over ranks."""
    for _ in range(warmup):
        step()
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    t0 = time.perf_counter()
    for _ in range(steps):
        step()
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    elapsed = time.perf_counter() - t0
    if world > 1:
        tmax = torch.tensor([elapsed], device="cuda", dtype=torch.float64)
        elapsed = float(_all_reduce(torch, dist, tmax, dist.ReduceOp.MAX).item())
    return elapsed / steps * 1e3


def av_batch(torch, n, seed, device):
    wav, masks = synth_batch(torch, n, seed, device)
    g = torch.Generator(device=device)
    g.manual_seed(seed + 17)
    return wav, masks, torch.randn(n, T_FRAMES, 136, generator=g, device=device)


def dp_train_block(torch, dist, models, ops, ap_mod, cfg, device, rank, world):
    """AV data-parallel training, gradients all-reduced over RCCL inside the backward pass.

    `check` -- three TF-Adam steps on a fixed seeded GLOBAL batch of 32 x world utterances (T = 250, config 4's per-GPU
    share), sharded by rank, through the production path (backend nccl = RCCL on the driver's node: per-layer
    asynchronous all-reduce buckets behind each layer's weight-gradient kernels, 1 / world inside the fused Adam).
    `ranks_bit_identical`: elementwise MAX and MIN over ranks of the int32 view of every rank's variables agree, i.e.
    all ranks hold the same bits.  Then rank 0 repeats the same global batch ALONE (parallel.solo(): no collective;
    its peers wait at a barrier), shard by shard at the ranks' batch size -- the same kernels, only the collective differs:
    `max_abs_diff_vs_single_process` must stay under `bar` = 2e-5 and the first step's summed gradient must agree (a bucket
    that was not reduced is off by a factor of world there; Adam's variables cannot show it).  The run at the whole global
    batch in one launch (other kernel families) is reported beside it, informational.  `max_abs_update` shows the three
    steps moved the weights by two orders of magnitude more.

    Timings, each the driver's way (barrier + synchronize on both sides, max over ranks), same keys at every N:
    `weak_32_per_gpu` (per-GPU batch fixed at 32: global 32 N -- what north_star's >= 0.85 scaling is claimed for) and
    `fixed_global_256` (BASELINE configs[3] read literally: per-GPU batch 256 / N -- latency-bound by construction, a
    step of 32 utterances costs a third of a step of 256).  `ms_per_step_no_collective` is the same
    per-GPU step with the all-reduce switched off (every rank on its own), so the price of the collective is visible."""
    from avsi_amd import parallel
    grouped = dist.is_initialized()          # world > 1, or the one-rank rehearsal (AVSI_DP_REHEARSE=1)
    out = {"n_gpus": world, "backend": dist.get_backend() if grouped else None,
           "rccl_ranks": dist.get_world_size() if grouped else 1}
    if grouped and world == 1:
        out["rehearsal"] = ("one-rank %s communicator: bucketed asynchronous all-reduce, guard words, %d-CU cooperative "
                            "budget and 1 / world in the fused Adam all ran against it" % (dist.get_backend(), ops.coop_cu_budget()))

    # normalisation statistics from a seeded batch that is the same on every rank (the headline's are per-rank data)
    spec = ap_mod.frontend(synth_batch(torch, 64, 4242, device)[0], want_spec=True)['spec']
    mean, std = spec.mean(dim=(0, 1)), spec.std(dim=(0, 1), unbiased=False)
    del spec

    def build(n, w, m_, v, seed=11):
        seq = np.full(n, T_FRAMES)
        m = models.StackedBLSTMModel(seq, w, m_, mean, std, 0.0, dict(cfg, batch_size=n, rows_per_wg=0, precision='f32'),
                                     video_features=v, input='av', seed=seed, is_training=True)   # same weights on all ranks

        def step():
            m.feed(sequence_lengths=seq, target_sources=w, masks=m_, video_features=v)
            loss = m.loss_func
            m.train_op
            return loss
        return m, step

    # ---- (a) correctness self-check
    per = 32
    G = per * world
    wav, masks, video = av_batch(torch, G, 4242, device)          # the same seed, i.e. the same global batch, on every rank
    sl = slice(rank * per, (rank + 1) * per)

    out["coop_fallbacks"] = 0

    def fell_back(m):
        """True (after falling back to the batch-stationary kernels, in this process) when the step guard of `m`'s last
        step reports a cooperative-kernel timeout.  The guard words are summed over the ranks inside the last gradient
        bucket and the status word is sticky, so every rank of a data-parallel run takes the same branch; the updates of
        the void steps were skipped on the device.  The caller repeats the measurement."""
        if float(m.step_guard[1]) == 0.0:
            return False
        ops.coop_fall_back(device)
        out["coop_fallbacks"] += 1
        return True

    def three_steps(n, w, m_, v):
        for attempt in range(3):              # at most two fall-backs: tolerant cooperative kernels, then batch-stationary
            m, step = build(n, w, m_, v)
            init = m.variables.flat.clone()
            losses, g1 = [], None
            for i in range(3):
                losses.append(step())
                if i == 0:
                    g1 = m.gradients.clone()        # after train_op: the gradient the update used, SUMMED over the ranks
            losses = torch.stack(losses)
            if not fell_back(m):
                break
        ops.coop_check(device)
        return m.variables.flat.clone(), init, losses, g1

    def three_steps_in_shards(n, shards, w, m_, v):
        """The like-with-like reference: ONE process takes the same three steps shard by shard (parallel.shards_step) --
        every shard at the ranks' batch size, i.e. on the kernels the ranks ran -- sums the gradients in rank order and
        applies them with 1 / shards.  Only the collective differs from the data-parallel run."""
        seq = np.full(n, T_FRAMES)
        feeds = [dict(sequence_lengths=seq, target_sources=w[r * n:(r + 1) * n].contiguous(),
                      masks=m_[r * n:(r + 1) * n].contiguous(), video_features=v[r * n:(r + 1) * n].contiguous())
                 for r in range(shards)]
        for attempt in range(3):
            m, _ = build(n, feeds[0]['target_sources'], feeds[0]['masks'], feeds[0]['video_features'])
            losses, g1 = [], None
            for i in range(3):
                ls, gsum = parallel.shards_step(m, feeds)
                losses.append(torch.stack(ls).double().mean())
                if i == 0:
                    g1 = gsum.clone()
            if not fell_back(m):
                break
        ops.coop_check(device)
        return m.variables.flat.clone(), torch.stack(losses), g1

    flat, init, losses, g1 = three_steps(per, wav[sl].contiguous(), masks[sl].contiguous(), video[sl].contiguous())
    check = {"steps": 3, "per_gpu_batch": per, "global_batch": G, "frames": T_FRAMES,
             "max_abs_update": float((flat - init).abs().max())}
    if grouped:
        bits = flat.view(torch.int32)
        hi = _all_reduce(torch, dist, bits.clone(), dist.ReduceOp.MAX)
        lo = _all_reduce(torch, dist, bits.clone(), dist.ReduceOp.MIN)
        check["ranks_bit_identical"] = bool((hi == lo).all().item())
        mean_losses = _all_reduce(torch, dist, losses.double().clone(), dist.ReduceOp.SUM) / world
        # (ranks that SHARE a GPU -- the gloo rehearsals -- can starve each other's cooperative groups and fall back, each on its
        #  own: the ranks' kernel families may then differ from the ones rank 0 repeats the shards on, which is summation order again)
        levels = torch.tensor([float(ops.coop_level())], device=device)
        mixed = bool(_all_reduce(torch, dist, levels.clone(), dist.ReduceOp.MAX).item() !=
                     _all_reduce(torch, dist, levels.clone(), dist.ReduceOp.MIN).item())
        dist.barrier()
        if rank == 0:
            with parallel.solo():
                ref, ref_losses, ref_g1 = three_steps_in_shards(per, world, wav, masks, video)
                one, _, one_losses, _ = three_steps(G, wav, masks, video)
            # (1) THE GATE, like with like: the same three steps in one process, shard by shard at the ranks' batch size on
            # the ranks' kernels, gradients summed in rank order -- only the collective (and its order of adding the
            # ranks' terms) differs, so the variables agree to the last bits of the gradient sums
            check["max_abs_diff_vs_single_process"] = float((ref - flat).abs().max())
            check["bar"] = 2e-4 if mixed else 2e-5
            if mixed:
                check["bar_note"] = "the ranks ended on different fall-back levels (kernel families): summation order differs, bar 2e-4"

            check["loss_max_rel_diff_vs_single_process"] = float(((mean_losses - ref_losses.double()).abs()
                                                                  / ref_losses.double().abs()).max())
            # (2) the SUMMED gradient of the first step against the reference's sum.  Adam's update is (almost) invariant
            # to the scale of the gradient, so the variables above cannot see a bucket that was not reduced or was reduced
            # twice; the gradient buffer itself can: such a part is off by a factor of `world` (1 / world itself lives in
            # the fused Adam's grad_scale and, for the same reason, shows only through l2 > 0)
            scale = float(ref_g1.abs().max())
            check["first_step_summed_gradient_max_abs_diff_rel"] = float((g1 - ref_g1).abs().max()) / scale
            check["gradient_bar"] = 1e-4
            # (3) informational: one process at the whole global batch -- other recurrent kernel families above 64
            # utterances (another order of the 256-long sums; three Adam steps amplify the last bits of small gradients)
            check["max_abs_diff_vs_one_batch_of_%d" % G] = float((one - flat).abs().max())
            check["loss_max_rel_diff_vs_one_batch"] = float(((mean_losses - one_losses.double()).abs()
                                                             / one_losses.double().abs()).max())
            check["ok"] = bool(check["ranks_bit_identical"] and check["max_abs_diff_vs_single_process"] < check["bar"]
                               and check["first_step_summed_gradient_max_abs_diff_rel"] < check["gradient_bar"])
            del ref, one
        dist.barrier()
    else:
        check["note"] = "single process: nothing to compare (the N >= 2 runs of this bench carry the check)"
    check["coop_fallbacks_this_rank"] = out["coop_fallbacks"]
    out["check"] = check
    del wav, masks, video, flat, init

    # ---- (b) timings
    for key, per_b, scaling in (("weak_32_per_gpu", 32, "weak"), ("fixed_global_256", max(1, 256 // world), "strong")):
        w, m_, v = av_batch(torch, per_b, 8765 + rank, device)
        m, step = build(per_b, w, m_, v, seed=7)
        steps, warm = (30, 5) if per_b <= 64 else (12, 3)
        ms = time_steps_all_ranks(torch, dist, world, step, steps, warm)
        while fell_back(m):               # a residency conflict (e.g. with RCCL's kernels) costs a repetition, not the entry
            m, step = build(per_b, w, m_, v, seed=7)
            ms = time_steps_all_ranks(torch, dist, world, step, steps, warm)
        ops.coop_check(device)
        entry = {"workload": "configs[3] AV training step (front end + forward + BPTT + %sTF-Adam), %d utterances per GPU"
                             % ("RCCL gradient all-reduce + " if world > 1 else "", per_b),
                 "scaling": scaling, "per_gpu_batch": per_b, "global_batch": per_b * world, "ms_per_step": ms,
                 "value": per_b * world / ms * 1e3, "unit": "utterances/s"}
        entry["recurrent_kernels"] = ("default policy", "cooperative, splits <= 8 (fell back once)",
                                      "batch-stationary (fell back twice)")[ops.coop_level()]
        if grouped:
            with parallel.solo():
                entry["ms_per_step_no_collective"] = time_steps_all_ranks(torch, dist, world, step, steps, 2)
        out[key] = entry
        del m, step, w, m_, v
    return out


def named_workloads(torch, models, ops, model, cfg, mean, std, device, rank, world):
    """The sizes the reference and BASELINE.json name, next to the headline batch: inference on the 100 clips of
    configs[0/1] as ONE batch and at the reference's inference batch of 32 (scripts/inference.sh:7) -- plus 128 and 1024
    utterances, the mid sizes the round-1 review set targets for -- and the LWS phase reconstruction of 32 utterances.
    Each entry has its own ms_per_step.  (The AV training entries of configs[3] are `dp_train_block`.)"""
    out = {}
    for name, b in (("infer_b100", 100), ("infer_b32", 32), ("infer_b128", 128), ("infer_b1024", 1024)):
        wav, masks = synth_batch(torch, b, 4321 + rank, device)
        seq = np.full(b, T_FRAMES)
        m = models.StackedBLSTMModel(seq, wav, masks, mean, std, 0.0, dict(cfg, batch_size=b, rows_per_wg=0), input='a',
                                     is_training=False, variables=model.variables)

        def step(m=m, seq=seq, wav=wav, masks=masks):
            m.feed(sequence_lengths=seq, target_sources=wav, masks=masks)
            _ = m.prediction
            return m.loss_func
        # Ranks that SHARE a GPU (the gloo rehearsals of tests/: several processes, each wanting whole XCDs for its cooperative
        # groups) can starve each other into the bounded wait: fall back like the trainer and dp_train do and time the entry again
        # (at most twice: tolerant cooperative kernels, then batch-stationary).  One rank per GPU: never taken.
        for attempt in range(3):
            try:
                ms = time_steps(torch, step, 30 if b <= 128 else 10, 5 if b <= 128 else 3)
                ops.coop_check(device)
                break
            except ops.CoopTimeout:
                if attempt == 2 or ops.coop_level() >= 2:
                    raise
                ops.coop_fall_back(device)
                out["coop_fallbacks"] = out.get("coop_fallbacks", 0) + 1
        del m
        out[name] = {"workload": "configs[1] inference, %d utterances per step per GPU" % b, "per_gpu_batch": b,
                     "ms_per_step": ms, "value": b * world / ms * 1e3, "unit": "utterances/s"}
        if ops.coop_level():
            out[name]["recurrent_kernels"] = ("default policy", "cooperative, splits <= 8 (fell back once)",
                                              "batch-stationary (fell back twice)")[ops.coop_level()]
    # the step after the path in the reference's default `infer` (inference.py:141-154): LWS phase reconstruction of the
    # enhanced batch (STFT, 102 sweeps, stitching, inverse STFT) at the reference's inference batch of 32
    from avsi_amd import lws as lws_mod
    lb = 32
    lwav, lmask = lws_signal(torch, lb, 77 + rank, device)
    proc = lws_mod.lws(384, 192, fftsize=512, mode='speech')
    lms = time_steps(torch, lambda: proc.refine_enhanced(lwav, lmask, num_samples=N_SAMPLES), 5, 2)
    out["lws_b32"] = {"workload": "LWS phase reconstruction of 32 enhanced utterances (inference.py:141-154; harmonic "
                                  "test signal + noise, 33 gap frames)", "per_gpu_batch": lb, "ms_per_step": lms,
                      "value": lb * world / lms * 1e3, "unit": "utterances/s"}
    return out


def lws_signal(torch, n, seed, device):
    """Harmonic test signal + noise (what the LWS entries refine), one 33-frame gap."""
    gl = torch.Generator(device=device)
    gl.manual_seed(seed)
    tt = torch.arange(N_SAMPLES, device=device)[None, :].float()
    f0 = 150 + 100 * torch.rand(n, 1, generator=gl, device=device)
    w = sum(2000 / h * torch.sin(2 * np.pi * h * f0 * tt / 16000) for h in range(1, 9))
    w = w * (0.6 + 0.4 * torch.sin(2 * np.pi * 4 * tt / 16000)) + 100 * torch.randn(n, N_SAMPLES, generator=gl, device=device)
    m = torch.ones(n, T_FRAMES, 257, device=device)
    m[:, 100:133] = 0
    return w, m


def unet_setup(torch, models, ap_mod, B, seed, device, is_training=False):
    """configs[4] inputs and model: 1.024 s clips, 128 x 128 log-spectrogram, one whole-frame gap of 100 / 200 / 400 /
    800 ms at 8 ms frames (1600 ms exceeds the 0.8 coverage cap of a 1 s clip)."""
    N, T, F = 16384, 128, 128
    cfg = dict(audio_feat_dim=F, audio_len=N, net_dim=[H, H, H], optimizer_type='adam', starter_learning_rate=1e-3,
               lr_updating_steps=10000, lr_decay=1.0, batch_size=B, l2=0.0)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    wav = torch.clamp(torch.round(torch.randn(B, N, generator=g, device=device) * 3000.0), -32768, 32767)
    lens = torch.tensor([12, 25, 50, 100], device=device)[torch.randint(0, 4, (B,), generator=g, device=device)]
    starts = (torch.rand(B, generator=g, device=device) * (T - lens).float()).long()
    t = torch.arange(T, device=device)[None, :]
    masks = torch.ones(B, T, F, device=device)
    masks[(t >= starts[:, None]) & (t < (starts + lens)[:, None])] = 0.0
    spec = ap_mod.frontend(wav[:min(B, 256)], window_size=16, step_size=8, n_fft=256, num_bins=F, want_spec=True)['spec']
    mean, std = spec.mean(dim=(0, 1)), spec.std(dim=(0, 1), unbiased=False)
    seq = np.full(B, T)
    model = models.UNetFConvModel(seq, wav, masks, mean, std, 0.0, cfg, is_training=is_training, seed=7)

    def step():
        model.feed(sequence_lengths=seq, target_sources=wav, masks=masks)
        _ = model.prediction
        return model.loss_func
    return model, step


UNET_FLOPS_PER_CLIP = 0.52e9          # 2 k^2 Cin Cout H W over the 13 layers
AV_FWD_FLOPS = 2.207e9                # forward, AV model (D = 393), per utterance
AV_WGRAD_FLOPS = 2.0 * ((393 + 500 + 500) * 2000 * 250 + 6 * 250 * 1000 * 249 + 500 * 257 * 250)   # dWx + dWh + dW_proj
ISTFT_BYTES = 250 * 257 * 4 * 2 + 48000 * 4 + 48000 * 4          # prediction + mask + target waveform in, waveform out
ISTFT_BYTES_FROM_STFT = 250 * 257 * 4 * 2 + 250 * 257 * 8 + 48000 * 4     # round 3's form: complex target STFT in instead


def e2e_workloads(torch, device):
    """The reference's drivers end to end on GRID-sized records (one TFRecord file per utterance, as its datasets have them)
    under /dev/shm: `infer()` -- records in, int16 WAV files out: reading, parsing, upload, network, waveform reconstruction,
    (LWS phase refinement,) read-back and file writing (inference.py:121-170) -- and `train()` (training_emb.py:214-363:
    reading, parsing, upload, step, loss bookkeeping; the per-step figure is the time inside an epoch).  What a drop-in user
    of `speech_inpainting_main.py inference / training` gets from one GPU, next to the resident-input kernel rates above."""
    import contextlib
    import io
    import re
    import shutil
    import struct
    import tempfile
    from avsi_amd import inference, training, tfrecord_io as tio
    from avsi_amd.config_utils import check_trainconfiguration, load_configfile
    out = {}
    base = tempfile.mkdtemp(prefix='avsi_bench_e2e_', dir='/dev/shm' if os.path.isdir('/dev/shm') else None)
    try:
        n_infer, n_train = 16384, 2048
        rng = np.random.default_rng(0)
        wav = np.round(rng.normal(0, 3000, N_SAMPLES)).astype(np.float32)
        mask = np.ones((T_FRAMES, F_BINS), np.float32)
        mask[100:100 + GAP_FRAMES] = 0
        video = rng.normal(size=(T_FRAMES, 136)).astype(np.float32)
        # one record, serialised once; every file gets its own sample path (same length) and checksum
        tag = b"clip_0000000"
        payload = bytearray(tio.serialize_sample_fixed(T_FRAMES, 20, wav, video, mask, np.zeros(50, np.float32), tag.decode()))
        at = bytes(payload).index(tag)
        head = struct.pack('<Q', len(payload))
        head += struct.pack('<I', tio.masked_crc32c(head))
        root = os.path.join(base, "data", "test-set")
        os.makedirs(root)
        t0 = time.perf_counter()
        for i in range(n_infer):
            payload[at:at + len(tag)] = b"clip_%07d" % i
            body = bytes(payload)
            with open(os.path.join(root, "data_%05d.tfrecord" % (i + 1)), 'wb') as fh:
                fh.write(head + body + struct.pack('<I', tio.masked_crc32c(body)))
        for name, n in (("training-set", n_train), ("validation-set", 64)):
            d = os.path.join(base, "data", name)
            os.makedirs(d)
            for i in range(n):
                os.link(os.path.join(root, "data_%05d.tfrecord" % (i + 1)), os.path.join(d, "data_%05d.tfrecord" % (i + 1)))
            np.save(os.path.join(d, "seq_lengths.npy"), np.full(n, T_FRAMES))
        t_write = time.perf_counter() - t0
        net = os.path.join(base, "logs", "exp", "netmodel")
        os.makedirs(net)
        np.save(os.path.join(base, "mean.npy"), np.zeros(F_BINS))
        np.save(os.path.join(base, "std.npy"), np.full(F_BINS, 3.0))
        cfg_lines = ["model = av-blstm", "audio_feat_dim = 257", "video_feat_dim = 136", "audio_len = %d" % N_SAMPLES,
                     "batch_size = 32", "net_dim = [250, 250, 250]", "dropout_rate = 0.0", "max_n_epochs = 2",
                     "n_earlystop_epochs = 5", "optimizer_type = adam", "starter_learning_rate = 0.001", "lr_decay = 1.0",
                     "lr_updating_steps = 10000", "l2 = 0.0", "num_asr_labels = 33", "ctc_loss = 0.001", "learning_rate = 0.001",
                     "integration_layer = 0", "root_folder = %s" % os.path.join(base, "data"),
                     "exp_folder = %s" % os.path.join(base, "logs", "exp"), "device = /gpu:0",
                     "audio_feat_mean = %s" % os.path.join(base, "mean.npy"), "audio_feat_std = %s" % os.path.join(base, "std.npy"), ""]
        cfg_file = os.path.join(base, "train.config")
        open(cfg_file, "w").write("\n".join(cfg_lines))

        # ---- train(): two epochs of 64 steps of 32 utterances (configs[3]'s per-GPU share), then its checkpoint serves infer()
        buf = io.StringIO()
        t0 = time.perf_counter()
        with contextlib.redirect_stdout(buf):
            training.train(cfg_file)
        t_train = time.perf_counter() - t0
        epochs = [float(x) for x in re.findall(r"Epoch training time \(seconds\) = ([0-9.]+)", buf.getvalue())]
        steps = n_train // 32
        out["e2e_train_b32"] = {
            "workload": "training.train() end to end on %d GRID-sized TFRecord files under /dev/shm, batch 32: ms per step INSIDE an "
                        "epoch (reading, parsing, upload, step, loss bookkeeping), best epoch of %d" % (n_train, len(epochs)),
            "per_gpu_batch": 32, "ms_per_step": min(epochs) / steps * 1e3, "value": 32 * steps / min(epochs), "unit": "utterances/s",
            "whole_call_s": t_train, "epochs_s": epochs}

        def run_infer(n, batch, oracle_phase, tag_, coalesce=None):
            sub = os.path.join(base, "sub_%s" % tag_)
            os.makedirs(sub)
            for i in range(n):
                os.link(os.path.join(root, "data_%05d.tfrecord" % (i + 1)), os.path.join(sub, "data_%05d.tfrecord" % (i + 1)))
            best = None
            before = os.environ.get('AVSI_INFER_COALESCE')
            if coalesce is not None:
                os.environ['AVSI_INFER_COALESCE'] = str(coalesce)
            try:
                for rep in range(2):
                    t0_ = time.perf_counter()
                    with contextlib.redirect_stdout(io.StringIO()):
                        inference.infer(net, sub, os.path.join(base, "audio_%s_%d" % (tag_, rep)), "enh", norm=True,
                                        oracle_phase=oracle_phase, batch_size=batch)
                    dt = time.perf_counter() - t0_
                    best = dt if best is None else min(best, dt)
                    shutil.rmtree(os.path.join(base, "audio_%s_%d" % (tag_, rep)), ignore_errors=True)
            finally:
                if coalesce is not None:
                    if before is None:
                        os.environ.pop('AVSI_INFER_COALESCE', None)
                    else:
                        os.environ['AVSI_INFER_COALESCE'] = before
            how = ("one model step per reader batch (AVSI_INFER_COALESCE=0: the reference's sess.run granularity)" if coalesce == 0 else
                   "the driver's default: the model steps of up to 1024 utterances' reader batches run as one launch sequence "
                   "(utterances are independent; files, per-batch lines and per-batch losses as with one step per batch)")
            return {"workload": "inference.infer() end to end: %d TFRecord files -> int16 WAV files under /dev/shm, batch_size %d, %s; %s; "
                                "whole call including model construction and checkpoint restore, best of 2" % (
                                    n, batch, "oracle phase" if oracle_phase else "LWS phase refinement (the reference's default)", how),
                    "per_gpu_batch": batch, "utterances": n, "seconds": best, "ms_per_step": best / (n / batch) * 1e3,
                    "value": n / best, "unit": "utterances/s"}
        out["e2e_infer_b1024_oracle_phase"] = run_infer(n_infer, 1024, True, "o1024")
        out["e2e_infer_b1024"] = run_infer(n_infer, 1024, False, "l1024")
        out["e2e_infer_b32_oracle_phase"] = run_infer(4096, 32, True, "o32")
        out["e2e_infer_b32"] = run_infer(4096, 32, False, "l32")
        out["e2e_infer_b32_oracle_phase_step_per_batch"] = run_infer(4096, 32, True, "o32s", coalesce=0)
        out["e2e_infer_b32_step_per_batch"] = run_infer(4096, 32, False, "l32s", coalesce=0)
        out["e2e_dataset"] = {"files": n_infer, "bytes_per_file": len(payload) + 16, "written_in_s": t_write, "where": base.rsplit('/', 1)[0]}
    finally:
        shutil.rmtree(base, ignore_errors=True)
    return out


def extra_workloads(torch, models, ops, ap_mod, cfg, mean, std, device):
    """N = 1 only: the other configurations of BASELINE.json and the steps either side of the path, each with its own
    ms_per_step and an ALGORITHMIC (unpadded) roofline figure: AV training at 8192 utterances, the U-Net at
    512 and at the reference's batch of 32, the fused inverse STFT at 4096 utterances (row f1), LWS phase
    reconstruction at 1024 (row a14 / f4), and the headline step fed from pinned host arrays at the reference's feed
    boundary (training.py:67-74), which states the PCIe-inclusive rate."""
    out = {}

    def guarded(name, fn):
        t0 = time.perf_counter()
        try:
            out[name] = fn()
        except Exception as e:        # an entry that fails says so; the others still run
            out[name] = {"error": "%s: %s" % (type(e).__name__, str(e)[:300])}
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        print("[bench] %s: %.0f s" % (name, time.perf_counter() - t0), file=sys.stderr, flush=True)

    def train_b8192():
        B = 8192
        wav, masks, video = av_batch(torch, B, 99, device)
        seq = np.full(B, T_FRAMES)
        timer = KernelTimer(torch)
        plain = {n: getattr(ops, n) for n in ("blstm_rec_bwd", "gemm_splitk")}
        for n, fn in plain.items():
            setattr(ops, n, timer.wrap(n, fn))
        try:
            m = models.StackedBLSTMModel(seq, wav, masks, mean, std, 0.0, dict(cfg, batch_size=B, rows_per_wg=0, precision='f32'),
                                         video_features=video, input='av', seed=7, is_training=True)

            def step():
                m.feed(sequence_lengths=seq, target_sources=wav, masks=masks, video_features=video)
                loss = m.loss_func
                m.train_op
                return loss
            step()
            timer.reset(2, 1)
            ms = time_steps(torch, step, 2, 0)
            ops.coop_check(device)
            tot = timer.totals()
        finally:
            for n, fn in plain.items():
                setattr(ops, n, fn)
        # the two recurrent kernels of training ALONE on resident operands of the same shape (tools/rec_bwd_time.py,
        # tools/rec_fwd_time.py): inside the step they share the chip with the side streams' kernels
        del m
        torch.cuda.empty_cache()
        alone = {}
        from avsi_amd import _lib as _l
        bwd_name = _l.lib().avsi_blstm_rec_bwd_kernel_name(B).decode()      # what the BPTT entry launches at this batch
        try:
            def timed(fn):
                for _ in range(2):
                    fn()
                e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                e0.record()
                for _ in range(3):
                    fn()
                e1.record()
                torch.cuda.synchronize()
                t = e0.elapsed_time(e1) / 3
                tf = 0.25e9 * B / (t * 1e-3) / 1e12
                return {"ms": t, "TFLOP/s": tf, "frac": tf / FP32_MFMA_PEAK_TFLOPS}
            resv = torch.rand(T_FRAMES, B, 2, 5, 256, device=device) * 0.9 + 0.05
            wts = torch.randn(2 * 262144, device=device) * 0.05
            dh = torch.randn(T_FRAMES, B, 512, device=device)
            dz = torch.empty(T_FRAMES, B, 2048, device=device)
            alone[bwd_name] = timed(lambda: plain["blstm_rec_bwd"](dh, resv, wts, dz, split=0))
            dz.normal_(0.0, 0.3)
            alone["blstm_rec_fwd_pp_kernel<true> (with reserve)"] = timed(lambda: ops.blstm_rec_fwd(dz, wts, dh, resv, split=0))
            alone["blstm_rec_fwd_pp_kernel<false>"] = timed(lambda: ops.blstm_rec_fwd(dz, wts, dh, None, split=0))
            del resv, wts, dh, dz
        except Exception as e:
            alone["error"] = "%s: %s" % (type(e).__name__, str(e)[:200])
        t_bwd, n_bwd = tot["blstm_rec_bwd"]
        t_wg, _ = tot["gemm_splitk"]
        bwd_tf = 0.25e9 * B * n_bwd / (t_bwd * 1e-3) / 1e12
        wg_tf = AV_WGRAD_FLOPS * B * 2 / (t_wg * 1e-3) / 1e12
        return {"workload": "configs[2]: AV 3xBLSTM-250 training step (front end + forward + BPTT + TF-Adam), 8192 utterances",
                "per_gpu_batch": B, "ms_per_step": ms, "value": B / ms * 1e3, "unit": "utterances/s",
                "algorithmic_TFLOP/s": 3 * AV_FWD_FLOPS * B / (ms * 1e-3) / 1e12,
                "frac_of_fp32_mfma_peak": 3 * AV_FWD_FLOPS * B / (ms * 1e-3) / 1e12 / FP32_MFMA_PEAK_TFLOPS,
                "kernels_alone": alone,
                "kernels": {bwd_name: {"avg_launch_ms": t_bwd / n_bwd, "TFLOP/s": bwd_tf,
                                                        "frac": bwd_tf / FP32_MFMA_PEAK_TFLOPS},
                            "gemm_dma_kernel<true,...> (weight gradients, split-K A^T.B)": {
                                "ms_per_step": t_wg / 2, "TFLOP/s": wg_tf, "frac": wg_tf / FP32_MFMA_PEAK_TFLOPS}}}
    guarded("train_b8192", train_b8192)

    def unet(B, steps, warm):
        def run():
            m, step = unet_setup(torch, models, ap_mod, B, 4321, device)
            ms = time_steps(torch, step, steps, warm)
            tf = UNET_FLOPS_PER_CLIP * B / (ms * 1e-3) / 1e12
            return {"workload": "configs[4]: U-Net (fconv) spectrogram inpainter, inference, %d clips per step" % B,
                    "per_gpu_batch": B, "ms_per_step": ms, "value": B / ms * 1e3, "unit": "clips/s",
                    "algorithmic_TFLOP/s": tf, "frac_of_fp32_mfma_peak": tf / FP32_MFMA_PEAK_TFLOPS}
        return run
    guarded("unet_b512", unet(512, 10, 3))
    guarded("unet_b32", unet(32, 30, 5))

    def unet_train(B, steps, warm):
        def run():
            m, _ = unet_setup(torch, models, ap_mod, B, 4321, device, is_training=True)
            seq, wav, masks = m.sequence_lengths, m.target_sources, m.masks

            def step():
                m.feed(sequence_lengths=seq, target_sources=wav, masks=masks)
                loss = m.loss_func
                m.train_op
                return loss
            ms = time_steps(torch, step, steps, warm)
            tf = 3.0 * UNET_FLOPS_PER_CLIP * B / (ms * 1e-3) / 1e12
            return {"workload": "configs[4]: U-Net training step (front end + forward + backward + TF-Adam, models.py:688-702), "
                                "%d clips per step" % B, "per_gpu_batch": B, "ms_per_step": ms, "value": B / ms * 1e3,
                    "unit": "clips/s", "algorithmic_TFLOP/s": tf, "frac_of_fp32_mfma_peak": tf / FP32_MFMA_PEAK_TFLOPS,
                    "algorithmic_flops_per_clip": 3.0 * UNET_FLOPS_PER_CLIP}
        return run
    guarded("unet_train_b512", unet_train(512, 6, 2))
    guarded("unet_train_b32", unet_train(32, 20, 4))

    def istft_b4096():
        B = 4096
        wav, masks = synth_batch(torch, B, 555, device)
        fe = ap_mod.frontend(wav, want_spec=True, want_stft=True)
        pred, stft = fe['spec'], fe['stft']
        zero, one = torch.zeros(F_BINS, device=device), torch.ones(F_BINS, device=device)
        ms = time_steps(torch, lambda: ap_mod.enhanced_from_prediction_wav(pred, zero, one, wav, masks, num_samples=N_SAMPLES), 10, 3)
        ms2 = time_steps(torch, lambda: ap_mod.enhanced_from_prediction(pred, zero, one, stft, masks, num_samples=N_SAMPLES), 10, 3)
        gbs, gbs2 = ISTFT_BYTES * B / (ms * 1e-3) / 1e9, ISTFT_BYTES_FROM_STFT * B / (ms2 * 1e-3) / 1e9
        return {"workload": "row f1: enhanced_sources (exp(pred std + mean), phase of the masked target -- its STFT taken "
                            "inside the kernel from the target waveform --, inverse STFT, models.py:181-197), 4096 utterances",
                "per_gpu_batch": B, "ms_per_step": ms,
                "value": B / ms * 1e3, "unit": "utterances/s", "GB/s": gbs, "frac_of_hbm_peak": gbs / HBM_PEAK_GBS,
                "algorithmic_bytes_per_utterance": ISTFT_BYTES,
                "from_stored_stft": {"ms_per_step": ms2, "GB/s": gbs2, "frac_of_hbm_peak": gbs2 / HBM_PEAK_GBS,
                                     "algorithmic_bytes_per_utterance": ISTFT_BYTES_FROM_STFT,
                                     "note": "round 3's form (mode 2): reads the 514 kB complex STFT the front end had to write"}}
    guarded("istft_b4096", istft_b4096)

    def lws_b1024():
        from avsi_amd import lws as lws_mod
        B = 1024
        w, m = lws_signal(torch, B, 78, device)
        proc = lws_mod.lws(384, 192, fftsize=512, mode='speech')
        ms = time_steps(torch, lambda: proc.refine_enhanced(w, m, num_samples=N_SAMPLES), 2, 1)
        # algorithmic work of the sweeps (what bounds them is vector-instruction issue): 102 sweeps x 252 frames x
        # 257 bins x 31 complex multiply-adds (8 flop) + the rotation, norm and scale of a bin (~30 flop)
        gflop = 102 * 252 * 257 * (31 * 8 + 30) / 1e9
        return {"workload": "LWS phase reconstruction of 1024 enhanced utterances (inference.py:141-154)", "per_gpu_batch": B,
                "ms_per_step": ms, "value": B / ms * 1e3, "unit": "utterances/s", "kernel": proc.kernel_for(B),
                "algorithmic_GFLOP_per_utterance": gflop, "algorithmic_TFLOP/s": gflop * B / ms,
                "frac_of_fp32_vector_peak": gflop * B / ms / 157.3}
    guarded("lws_b1024", lws_b1024)

    def infer_b8192_hostfed():
        # the reference's feed boundary hands over HOST arrays (feed_dict, training.py:67-74): wav 1.57 GB + masks 2.1 GB per
        # step of 8192.  Pinned host memory, uploaded on a copy stream into the buffer set the NEXT step computes on
        # (double-buffered: the upload of step i + 1 runs under the kernels of step i); `serial` = upload, then compute.
        B = 8192
        wav_d, masks_d = synth_batch(torch, B, 1234, device)
        wav_h = torch.empty(wav_d.shape, dtype=torch.float32, pin_memory=True).copy_(wav_d)
        masks_h = torch.empty(masks_d.shape, dtype=torch.float32, pin_memory=True).copy_(masks_d)
        sets = [(wav_d, masks_d), (torch.empty_like(wav_d), torch.empty_like(masks_d))]
        seq = np.full(B, T_FRAMES)
        m = models.StackedBLSTMModel(seq, wav_d, masks_d, mean, std, 0.0, dict(cfg, batch_size=B, rows_per_wg=0, precision='f32'),
                                     input='a', seed=7, is_training=False)
        # a HIGH-PRIORITY stream: HIP multiplexes its streams onto four hardware queues per priority level, and by now
        # this process has created enough streams that the next normal one shares the queue of the launch stream -- its
        # copies and their event waits then sit IN ORDER between the step's kernels and nothing overlaps (measured:
        # 207 ms instead of 140, tools/hostfed_probe.py); queues of another priority are never shared with it
        copy = torch.cuda.Stream(device=device, priority=-1)
        main = torch.cuda.current_stream(device)
        state = {"i": 0, "ready": None}

        def upload(into):
            copy.wait_stream(main)                  # the set being overwritten was last read two steps ago on `main`
            with torch.cuda.stream(copy):
                into[0].copy_(wav_h, non_blocking=True)
                into[1].copy_(masks_h, non_blocking=True)
                ev = torch.cuda.Event()
                ev.record(copy)
            return ev

        def step_overlapped():
            cur = sets[state["i"] % 2]
            if state["ready"] is not None:
                main.wait_event(state["ready"])
            state["ready"] = upload(sets[(state["i"] + 1) % 2])
            m.feed(sequence_lengths=seq, target_sources=cur[0], masks=cur[1])
            _ = m.prediction
            state["i"] += 1
            return m.loss_func

        def step_serial():
            main.wait_event(upload(sets[0]))
            m.feed(sequence_lengths=seq, target_sources=sets[0][0], masks=sets[0][1])
            _ = m.prediction
            return m.loss_func
        ms = time_steps(torch, step_overlapped, 5, 2)
        ms_serial = time_steps(torch, step_serial, 3, 1)
        nbytes = wav_h.numel() * 4 + masks_h.numel() * 4
        return {"workload": "configs[1] inference step of 8192 utterances, inputs arriving as pinned host arrays at the reference's "
                            "feed boundary (training.py:67-74): PCIe-inclusive", "per_gpu_batch": B, "ms_per_step": ms,
                "value": B / ms * 1e3, "unit": "utterances/s", "host_bytes_per_step": nbytes,
                "serial_upload_then_compute": {"ms_per_step": ms_serial, "value": B / ms_serial * 1e3}}
    guarded("infer_b8192_hostfed", infer_b8192_hostfed)
    return out


def free_port():
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def self_launch(n):
    """`python bench.py --gpus N` without a launcher around it: start `python -m torch.distributed.run --nnodes=1
    --nproc-per-node N --master-addr 127.0.0.1 --master-port <free> bench.py <the same arguments>` as a CHILD process (same
    process group), pass its stdout (rank 0's one JSON line) and stderr through, forward SIGTERM / SIGINT to the launcher,
    and return its exit status.  Called before this process imports torch: it never initialises a GPU."""
    import signal
    import subprocess
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", str(n), "--master-addr",
           "127.0.0.1", "--master-port", str(free_port()), os.path.abspath(__file__)] + sys.argv[1:]
    env = dict(os.environ)
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")      # dmabuf IPC: RCCL's intra-node transport needs it on this image
    env.setdefault("OMP_NUM_THREADS", "1")
    # (same process group as this process: whoever stops the bench by its group -- a driver's timeout -- stops the ranks too)
    child = subprocess.Popen(cmd, env=env)

    def forward(signum, _frame):          # the launcher passes SIGTERM / SIGINT on to its workers
        try:
            child.send_signal(signum)
        except ProcessLookupError:
            pass
    for sig in (signal.SIGTERM, signal.SIGINT):
        signal.signal(sig, forward)
    rc = child.wait()
    return rc if rc >= 0 else 128 - rc


def timed_steps(torch, dist, ops, timer, step, steps, warmup, world, shared, device):
    """(seconds, loss of the last step, fall-backs): `warmup` untimed steps, then exactly `steps` between barriers; the time is the
    largest over the ranks.

    Ranks that SHARE a GPU (`shared`) can starve each other's cooperative groups into the bounded wait (see the named workloads): then
    every rank takes the fall-back together and the whole measurement is made again, at most twice.  With a GPU of its own for each
    rank the first attempt is the only one, and a timeout ends the run."""
    on = device if world > 1 and dist.get_backend() == "nccl" else "cpu"

    def largest(value, dtype):
        if world > 1:
            value = torch.tensor([value], device=on, dtype=dtype)
            dist.all_reduce(value, op=dist.ReduceOp.MAX)
            value = value.item()
        return value

    polls, ops.COOP_POLL_RAISES = ops.COOP_POLL_RAISES, ops.COOP_POLL_RAISES and not shared
    try:
        for fallbacks in range(3):
            for _ in range(warmup):
                step()
            timer.reset(steps, warmup)
            if world > 1:
                dist.barrier()
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            for _ in range(steps):
                loss = step()
            torch.cuda.synchronize()
            if world > 1:
                dist.barrier()
            elapsed = largest(time.perf_counter() - t0, torch.float64)
            loss = float(loss)
            try:
                ops.coop_check(device)
                late = 0
            except ops.CoopTimeout:
                if not shared:
                    raise
                late = 1
            if not (largest(late, torch.int32) if shared else 0):
                return elapsed, loss, fallbacks
            if fallbacks < 2:
                ops.coop_fall_back(device)
        raise ops.CoopTimeout(ops._COOP_MSG)
    finally:
        ops.COOP_POLL_RAISES = polls


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--batch", type=int, default=8192, help="utterances per GPU per step")
    ap.add_argument("--rows-per-wg", type=int, default=0)
    ap.add_argument("--cpu-sample", type=int, default=384, help="utterances timed on the CPU oracle (~15 s)")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--precision", choices=["f32", "bf16x3"], default="f32",
                    help="EXPLORATORY, inference only: bf16x3 = layer input projections with split-bf16 operands (hi.hi + hi.lo "
                         "+ lo.hi on the bf16 matrix cores, fp32 accumulation); never the default, never the headline")
    ap.add_argument("--no-also", action="store_true", help="skip the named-workload entries (`also` block: inference at 100, 32, 128 and 1024 utterances, training and LWS phase reconstruction at 32)")
    ap.add_argument("--also-timeout", type=int, default=420)
    ap.add_argument("--mode", choices=["infer", "train", "unet", "e2e"], default="infer",
                    help="infer = headline workload (configs[1]); train = configs[2]: AV model, fwd + BPTT + Adam; "
                         "unet = configs[4]: U-Net spectrogram inpainter inference (use --batch 32 .. 512)")
    args = ap.parse_args()
    t_bench0 = time.perf_counter()
    if args.gpus > 1 and "WORLD_SIZE" not in os.environ and "RANK" not in os.environ:
        # plain `python bench.py --gpus N`, the form the driver uses at N = 1: this process becomes the launcher of N ranks
        # (a CHILD torch.distributed.run; nothing here has imported torch or touched a GPU, and nothing is exec'ed)
        sys.exit(self_launch(args.gpus))

    import torch
    import torch.distributed as dist
    import avsi_amd  # noqa: F401
    from avsi_amd import models, ops

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    if args.gpus != world:
        sys.exit("bench.py --gpus %d inside a launch of %d ranks (WORLD_SIZE): the two must agree" % (args.gpus, world))
    local_rank %= torch.cuda.device_count()        # ranks sharing a GPU (gloo rehearsal) all map onto it
    torch.cuda.set_device(local_rank)
    device = torch.device("cuda", local_rank)
    from avsi_amd import parallel
    if world > 1 or parallel.rehearsing():
        # AVSI_DP_REHEARSE=1 at N = 1: a one-rank RCCL communicator, so that `dp_train` runs the bucketed asynchronous
        # all-reduce, the guard words and the CU reserve against RCCL's stream on a one-GPU box (parallel.rehearsing)
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        # a private free port only for the one-rank rehearsal: the ranks of a real job must agree on ONE port, so it comes
        # from the launcher (torch.distributed.run exports it) or is the fixed default parallel.init uses as well
        os.environ.setdefault("MASTER_PORT", str(free_port()) if world == 1 else "29500")
        # RCCL (backend "nccl") in production; AVSI_DIST_BACKEND=gloo lets several ranks share one GPU to rehearse
        # the multi-rank path on a single-GPU box (tests/test_bench_contract_gpu.py)
        backend = os.environ.get("AVSI_DIST_BACKEND", "nccl")
        if backend == "nccl":
            dist.init_process_group("nccl", rank=rank, world_size=world, device_id=device)
        else:
            dist.init_process_group(backend, rank=rank, world_size=world)

    if args.mode == "unet":
        return bench_unet(args, torch, dist, rank, world, device)
    if args.mode == "e2e":          # the drivers end to end, one JSON object (the `also.e2e_*` entries of the default line)
        torch.set_num_threads(1)
        print(json.dumps(e2e_workloads(torch, device)))
        return

    B = args.batch
    cfg = dict(audio_feat_dim=F_BINS, video_feat_dim=136, audio_len=N_SAMPLES, net_dim=[H, H, H],
               optimizer_type='adam', starter_learning_rate=1e-3, lr_updating_steps=10000, lr_decay=1.0,
               batch_size=B, l2=0.0, rows_per_wg=args.rows_per_wg, precision=args.precision)
    wav, masks = synth_batch(torch, B, 1234 + rank, device)
    # per-bin statistics of the synthetic set (restated compute_mean_std_features, type='spec')
    from avsi_amd import audio_processing as ap_mod
    spec = ap_mod.frontend(wav[:min(B, 256)], want_spec=True)['spec']
    mean = spec.mean(dim=(0, 1))
    std = spec.std(dim=(0, 1), unbiased=False)
    del spec
    seq = np.full(B, T_FRAMES)
    train = args.mode == "train"
    video = None
    if train:
        gv = torch.Generator(device=device)
        gv.manual_seed(99 + rank)
        video = torch.randn(B, T_FRAMES, 136, generator=gv, device=device)
    model = models.StackedBLSTMModel(seq, wav, masks, mean, std, 0.0, cfg, video_features=video,
                                     input='av' if train else 'a', seed=7, is_training=train)   # same weights on all ranks

    timer = KernelTimer(torch)
    # the front end's events bracket the C entry point itself (one kernel launch), not the Python function around it
    # (argument marshalling, a 2.1 GB torch.empty): its GB/s is the figure north_star names, so nothing else is inside
    from avsi_amd import _lib
    clib = _lib.lib()
    untimed = (ops.gemm, ops.blstm_rec_fwd, clib.avsi_frontend_f32)
    ops.gemm = timer.wrap("gemm_dma_kernel", ops.gemm)
    if args.precision == "bf16x3":
        ops.gemm_bf16x3 = timer.wrap("gemm_bf16x3_kernel", ops.gemm_bf16x3)
    ops.blstm_rec_fwd = timer.wrap("blstm_rec_fwd_kernel", ops.blstm_rec_fwd)
    clib.avsi_frontend_f32 = timer.wrap("frontend_kernel", clib.avsi_frontend_f32)
    if train:
        for name in ("blstm_rec_bwd", "gemm_splitk", "colsum", "adam_tf", "relayout_rows"):
            setattr(ops, name, timer.wrap(name, getattr(ops, name)))

    def step():
        model.feed(sequence_lengths=seq, target_sources=wav, masks=masks, video_features=video)
        if train:
            loss = model.loss_func
            model.train_op
            return loss
        _ = model.prediction
        return model.loss_func

    elapsed, loss_val, fallbacks = timed_steps(torch, dist, ops, timer, step, args.steps, args.warmup, world,
                                               world > torch.cuda.device_count(), device)
    totals = timer.totals()
    if rank == 0 and train:
        line = {"metric": "training utterances/sec (AV 3xBLSTM-250: front end + forward + BPTT + TF-Adam)",
                "value": B * world * args.steps / elapsed, "unit": "utterances/s", "n_gpus": world,
                "steps": args.steps, "warmup": args.warmup, "ms_per_step": elapsed / args.steps * 1e3,
                "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32", "data": "synthetic",
                "config": {"workload": "configs[2]: AV 3xBLSTM-250 training step", "per_gpu_batch": B,
                           "global_batch": B * world, "parallelism": "dp%d" % world},
                "loss_func": loss_val, "coop_fallbacks": fallbacks,
                "kernel_ms_per_step": {k: v[0] / args.steps for k, v in totals.items()},
                "calls_ms_last_step": {k: [round(s_.elapsed_time(e_), 2) for s_, e_ in v[-(len(v) // args.steps):]]
                                       for k, v in timer.events.items()}}
        print(json.dumps(line))
    if rank == 0 and not train:
        gemm_in, rec, proj = algorithmic_flops(B)
        t_rec, n_rec = totals["blstm_rec_fwd_kernel"]
        # ops.gemm is called 4 times per step: the three layer input projections -- one kernel symbol since round 6,
        # gemm_dma_kernel<false, false, 16, 3, false, 256, false, true> (wide tile, persistent workgroups), the dominant kernel: the
        # roofline block covers its three launches, as rocprofv3 --stats averages them -- and the 257-bin output projection
        # on <..., 256, true, true> (the same tile with the 257th bin folded in: a symbol of its own, in `others`).
        # AVSI_GEMM_FOLD_TAIL=0: 5 calls (256 bins on the wide tile + the last bin on a 32-wide tile); AVSI_PROJ_SPLIT=0 on top:
        # 4 calls, the projection on five 64-wide tiles
        ev = timer.events["gemm_dma_kernel"]
        per_step = len(ev) // args.steps
        ms = [s_.elapsed_time(e_) for s_, e_ in ev]
        folded = per_step == 4 and os.environ.get('AVSI_GEMM_FOLD_TAIL', '1') != '0'
        if args.precision == "bf16x3":      # exploratory: the layer projections are the split-bf16 launches
            layer_ms = [s_.elapsed_time(e_) for s_, e_ in timer.events["gemm_bf16x3_kernel"]]
            proj_ms, wide_proj_ms = ms, []
        else:
            layer_ms = [t for i, t in enumerate(ms) if i % per_step < 3]
            proj_ms = [t for i, t in enumerate(ms) if i % per_step >= 3]
            wide_proj_ms = [t for i, t in enumerate(ms) if i % per_step == 3] if (per_step == 5 or folded) else []
        t_layer = sum(layer_ms)
        t_gemm, n_gemm = t_layer, len(layer_ms)
        t_proj = sum(proj_ms)
        t_fe, n_fe = totals["frontend_kernel"]
        fe_ms = sorted(s_.elapsed_time(e_) for s_, e_ in timer.events["frontend_kernel"])
        rec_tf = rec * n_rec / (t_rec * 1e-3) / 1e12
        layer_tf = sum(gemm_in) * args.steps / (t_layer * 1e-3) / 1e12
        gemm_tf = layer_tf
        proj_tf = proj * args.steps / (t_proj * 1e-3) / 1e12
        fe_gbs = 706000.0 * B * n_fe / (t_fe * 1e-3) / 1e9
        if t_rec >= t_gemm:
            traffic, traffic_src = profiled_traffic("blstm_rec_fwd", B)
            roof = {"kernel": "blstm_rec_fwd_kernel", "bound": "mfma", "achieved": rec_tf,
                    "peak": FP32_MFMA_PEAK_TFLOPS, "unit": "TFLOP/s", "frac": rec_tf / FP32_MFMA_PEAK_TFLOPS,
                    "traffic": traffic, "traffic_source": traffic_src, "avg_launch_ms": t_rec / n_rec}
        else:
            traffic, traffic_src = profiled_traffic("gemm_dma_kernel", B)
            roof = {"kernel": "gemm_dma_kernel<false, false, 16, 3, false, 256, false, true>", "bound": "mfma", "achieved": gemm_tf,
                    "peak": FP32_MFMA_PEAK_TFLOPS, "unit": "TFLOP/s", "frac": gemm_tf / FP32_MFMA_PEAK_TFLOPS,
                    "traffic": traffic, "traffic_source": traffic_src, "avg_launch_ms": t_gemm / n_gemm}
        if args.precision == "bf16x3":
            roof["kernel"] = "gemm_bf16x3_kernel (EXPLORATORY: three bf16 MFMAs per fp32-equivalent product)"
            roof["peak"] = 2500.0 / 3.0      # dense bf16 MFMA peak (MI355X_MICROARCH.md) over the three products
            roof["frac"] = roof["achieved"] / roof["peak"]
            roof["traffic"], roof["traffic_source"] = None, None
        roof["others"] = {
            "blstm_rec_fwd_kernel": {"TFLOP/s": rec_tf, "ms_per_step": t_rec / args.steps},
            "gemm_dma_kernel(layer input projections)": {"TFLOP/s": layer_tf, "ms_per_step": t_layer / args.steps},
            "gemm_dma_kernel(257-bin projection: %s)" % (
                "one launch on the wide tile, the 257th bin folded in: gemm_dma_kernel<false, false, 16, 3, false, 256, true, true>"
                if folded else ("256 bins on the wide tile + 1 bin on a 32-wide tile" if wide_proj_ms else "64-wide tiles")):
                {"TFLOP/s": proj_tf, "ms_per_step": t_proj / args.steps},
            "frontend_kernel": {"GB/s": fe_gbs, "frac_of_hbm_peak": fe_gbs / HBM_PEAK_GBS,
                                "ms_per_step": t_fe / args.steps,
                                # one launch per step: spread over the timed steps, and the rate at the median launch
                                "launch_ms_min_median_max": [fe_ms[0], fe_ms[len(fe_ms) // 2], fe_ms[-1]],
                                "GB/s_at_median": 706000.0 * B / (fe_ms[len(fe_ms) // 2] * 1e-3) / 1e9,
                                "algorithmic_bytes_per_utterance": 706000,
                                # the model's call also writes the un-masked target spectrogram (257,000 B more per utterance) for the
                                # loss; with AVSI_LOSS_FROM_WAV=1 it stores the masked features only (its real traffic is then the
                                # algorithmic 706 kB) and the loss recomputes the target from the waveform -- slower overall
                                "writes_target_output": not model._loss_from_wav(),
                                "GB/s_real_traffic_at_median": (706000.0 if model._loss_from_wav() else 963000.0) * B
                                / (fe_ms[len(fe_ms) // 2] * 1e-3) / 1e9,
                                "device_copy_GB/s": device_copy_rate(torch, device),
                                "device_copy_GB/s_torch_copy_kernel": device_copy_rate(torch, device, kernel="torch")},
        }
        cpu, rms = (None, None)
        if rank == 0:
            print("[bench +%.0f s] headline timed; CPU baseline" % (time.perf_counter() - t_bench0), file=sys.stderr, flush=True)
        if not args.no_cpu_baseline and world == 1:     # the CPU leg is reported at N = 1 only
            sample = min(args.cpu_sample, B)
            # `model` still holds the results of the last TIMED step: its prediction rows are what gets checked
            pred_timed = model.prediction[:sample].cpu().numpy()
            cpu, rms = cpu_baseline(torch, model, wav, masks, mean, std, sample, pred_timed)
        line = {
            "metric": "masked utterances/sec (inference: front end + 3xBLSTM-250 forward + projection + L1 loss)",
            "value": B * world * args.steps / elapsed,
            "unit": "utterances/s",
            "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
            "ms_per_step": elapsed / args.steps * 1e3,
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
            "dtype": "f32" if args.precision == "f32" else "bf16x3 (layer input projections: split-bf16 operands, fp32 "
                                                             "accumulation; recurrence, projection, front end f32) -- EXPLORATORY",
            "data": "synthetic",
            "config": {"workload": "configs[1]: audio-only 3xBLSTM-250 inpainter, 3 s 16 kHz clips, one 400 ms gap, "
                                   "HIP STFT front end + fp32-MFMA BLSTM forward",
                       "per_gpu_batch": B, "global_batch": B * world, "frames": T_FRAMES, "parallelism": "dp%d" % world},
            "logmel_rms_vs_cpu_oracle": rms,
            "loss_func": loss_val, "coop_fallbacks": fallbacks,
            "roofline": roof,
            "cpu_baseline": cpu,
        }
    if not train and not args.no_also and args.precision == "f32":
        # Everything below runs AFTER the headline measurement is complete.  The dp_train block is the first code of this
        # repository to issue RCCL collectives from inside the backward pass on real multi-GPU hardware; a watchdog makes
        # sure a stall there cannot cost the headline line: when it fires, rank 0 prints the line it already has (with
        # the reason in `also`) and EVERY rank leaves with a non-zero status -- a hang must not read as a successful run.
        import threading
        progress = {"at": "start"}

        def mark(where):           # (stderr: the one JSON line on stdout stays alone; a long silent run reads as a hang)
            progress["at"] = where
            if rank == 0:
                print("[bench +%.0f s] %s" % (time.perf_counter() - t_bench0, where), file=sys.stderr, flush=True)
        if rank != 0:
            line = {}

        def give_up():
            if rank == 0:
                line.setdefault("also", {})["error"] = "named workloads did not finish within %d s (stalled in: %s)" % (
                    args.also_timeout, progress["at"])
                print(json.dumps(line), flush=True)
            os._exit(3)
        dog = threading.Timer(args.also_timeout, give_up)
        dog.daemon = True
        dog.start()
        ops.gemm, ops.blstm_rec_fwd, clib.avsi_frontend_f32 = untimed      # no per-call events in the small-batch entries
        torch.set_num_threads(1)       # launch-bound entries: no intra-op pool beside the launching thread (see cpu_baseline)
        variables = model.variables
        model._ws.clear()              # the headline's 40 GB of workspaces are not needed any more
        model._cache.clear()
        model.target_sources = model.masks = None
        del wav, masks
        torch.cuda.empty_cache()
        try:
            mark("dp_train")
            # on a high-priority stream, like training.train(): the steps' critical chain (cooperative recurrent kernels)
            # is then independent of which hardware queue the side streams and the collectives' stream happen to share,
            # and is dispatched ahead of them (tools/train_step_time.py: 6.3 .. 7.4 ms on the default stream depending on
            # the streams created before, 6.3 .. 6.6 on a high-priority one)
            hp = torch.cuda.Stream(device=device, priority=-1)
            hp.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(hp):
                dp = dp_train_block(torch, dist, models, ops, ap_mod, cfg, device, rank, world)
                hp.synchronize()
        except Exception as e:        # never a reason to lose the headline
            dp = {"error": "%s: %s" % (type(e).__name__, str(e)[:300])}
        line["dp_train"] = dp
        try:
            mark("also (inference at the named sizes, LWS at 32)")
            also = named_workloads(torch, models, ops, model, cfg, mean, std, device, rank, world)
            if "weak_32_per_gpu" in dp:
                also["train_b32"] = dp["weak_32_per_gpu"]
            if world == 1:
                mark("also (training at 8192, U-Net, inverse STFT, LWS at 1024, host-fed step)")
                also.update(extra_workloads(torch, models, ops, ap_mod, cfg, mean, std, device))
                mark("also (drivers end to end: train(), infer())")
                torch.cuda.empty_cache()
                try:
                    # in a child process of their own, as a user runs them (`speech_inpainting_main.py training / inference`):
                    # by now this process has created two dozen streams, and which hardware queue the trainer's streams
                    # share with them decides its step time (8.2 ms here against 6.7 in a fresh process)
                    import subprocess
                    # (a single-process run of the drivers: no rendezvous variables of this process in its environment)
                    env_e2e = {k: v for k, v in os.environ.items()
                               if k not in ("AVSI_DP_REHEARSE", "MASTER_PORT", "MASTER_ADDR", "RANK", "LOCAL_RANK", "WORLD_SIZE")}
                    child = subprocess.run([sys.executable, os.path.abspath(__file__), "--mode", "e2e"], capture_output=True,
                                           text=True, env=env_e2e, timeout=max(60, args.also_timeout - 120))
                    lines_ = [l for l in child.stdout.splitlines() if l.startswith("{")]
                    if child.returncode != 0 or not lines_:
                        raise RuntimeError("child exited with %d: %s" % (child.returncode, child.stderr[-300:]))
                    also.update(json.loads(lines_[-1]))
                except Exception as e:
                    also["e2e"] = {"error": "%s: %s" % (type(e).__name__, str(e)[:300])}
        except Exception as e:
            also = {"error": "%s: %s" % (type(e).__name__, str(e)[:300])}
        dog.cancel()
        line["also"] = also
    if rank == 0 and not train:
        print(json.dumps(line))
    if dist.is_initialized():
        dist.barrier()
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
