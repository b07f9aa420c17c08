"""Benchmark of the exact linear path on one MI355X.

    python bench.py [--gpus 1] [--steps K] [--warmup W] [--no-attention] [--no-decode-step] [--no-cpu]
    python bench.py --profile-kernel [--steps K]   (launches for rocprofv3 counter runs)
    python bench.py --profile-counters             (every sweep GEMM and attention shape, for counter runs)

Step: one pass of the decode-shaped exact linear sweep of a ~9B Qwen-style model (hidden
4096): QKV 4096->6144, O 4096->4096, gate_up 4096->24576 and down 12288->4096 at M in
{1, 16, 64, 256}, F = 14 truncated (3 INT8 dots, the enable() default), each through
the full exactmm::linear path (bf16 x -> digitize -> exact GEMM -> bf16 y). The step is a
HIP graph; weights rotate over copies so no use finds its weights in the MALL/L2; inputs
sit in HBM before timing starts. `value` is the sweep's algorithmic bytes
(2NK + 2MK + 2MN + 8N per linear) over the step time.

Also reported, from the same run:
* per-op times with GB/s, TOPS and roofline fractions, the hipBLASLt bf16 time and, for
  M > 16, the vendor int8 GEMM (torch._int_mm, one dot) on the same shape; `gemm_us` is the
  kernel the op runs without the digitize launch (the one-launch digitize + GEMM kernel at the
  row counts the table marks, `one_launch`);
* `roofline` of the dominant kernel (the GEMM launch with the largest share of the step),
  timed alone with HIP events on its own stream;
* split-bf16 paged decode attention at H=32/KV=8/D=128/BS=16 for 64x8K, 16x16K, 256x1K (TB/s);
* `lm_head`: the exact lm_head 4096->151936 at M = 16 and 256 with per-row activation scales
  10^U(-2,2) (full op time, roofline fractions, bit-exactness on sampled rows);
* `decode_step`: the synthetic decode step of the ~9B hybrid (32 layers of the four exact
  linears, paged attention on 8 of them, exact lm_head 4096->151936) at batch/context 256/1K,
  64/8K and 16/16K: ms per step as a HIP graph, the same step with hipBLASLt bf16 linears,
  for each leg the time of its linears, attention calls and glue each in a graph of its own,
  bitwise batch invariance of the logits, and a CPU estimate from the oracle's timings;
* bit-exactness against the CPU oracle: `bit_exact` on every per_op and per_op_f15 row
  (output rows 0..7, M/2 and M-1 of the op as timed), and on the line, all of them with
  lm_head's sampled rows and config 1's whole outputs (`bit_exact_scope` says which);
* `per_op_f15`: the 4-dot variant, the same sweep at F = 15 (offset digits) with the table
  tuned at F = 15, on weights packed at F = 15;
* `config1`: M = 16, K = N = 4096, F = 14 with all four dots and no split-K: GEMM and op
  times, and the whole fp32 and bf16 outputs checked bitwise against the oracle;
* `cpu_baseline`: the reference's CPU path (the torch int64 statements digitize_torch +
  exact_linear_torch) on every host thread (os.cpu_count() and torch.get_num_threads() are
  printed), config 1 in full and a bounded sample of the sweep's weight rows extrapolated per
  op; the C oracle (OpenMP) timed beside it as `oracle_c`.

The roofline's `traffic` is the HBM bytes per launch measured by rocprofv3 FETCH_SIZE and
WRITE_SIZE passes of `--profile-kernel` and recorded in profiles/; it is reported only when
that record was made on a library built from the current sources (`traffic_source` says which).
"""
import argparse
import json
import os
import sys
import time
from pathlib import Path

ROOT = Path(__file__).resolve().parent
sys.path.insert(0, str(ROOT / "vllm-exact_amd"))

METRIC = "exact GEMM INT8 TOPS (%MFMA peak) & GB/s (%HBM); decode-attn TB/s; bit-exact"
HBM_PEAK_GBS = 8000.0
INT8_PEAK_TOPS = 5000.0  # dense INT8 MFMA, MI355X published
SHAPES = [("qkv", 6144, 4096), ("o", 4096, 4096), ("gate_up", 24576, 4096), ("down", 4096, 12288)]
MS = [1, 16, 64, 256]
F, TRUNC, NDOTS = 14, True, 3
ATTN_CASES = [(64, 8192), (16, 16384), (256, 1024)]
DECODE_CASES = [(256, 1024), (64, 8192), (16, 16384)]  # (batch, context) of the decode-step emulation
HIDDEN, VOCAB, LAYERS, ATTN_EVERY, FFN = 4096, 151936, 32, 4, 12288
ATT_H, ATT_KV, ATT_D, ATT_BS = 32, 8, 128, 16


class DecodeStep:
    """Synthetic decode step of the ~9B hybrid with random-init weights (the GDN recurrence
    excluded): LAYERS layers of the four exact linears, paged decode attention on every
    ATTN_EVERY-th layer (8 of 32), and the exact lm_head. Non-attention layers pass the q
    slice of the QKV output on as the mixer output. Between linears: residual adds, SiLU-gated
    MLP, and a per-row power-of-two rescale (exact, so every op is row-local and batch
    invariant). `exact=False` runs the same step with hipBLASLt bf16 matmuls for the linears
    (same attention kernel): the non-exact baseline."""

    def __init__(self, torch, plugin, P, dev, gen, layers=LAYERS, vocab=VOCAB, keep_bf16=True):
        self.torch, self.P, self.dev = torch, P, dev
        self.layers = []
        for _ in range(layers):
            ws = {}
            for name, N, Kd in SHAPES:
                w = (torch.randn(N, Kd, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
                ws[name] = (plugin.pack_weight(w), w if keep_bf16 else None)
            self.layers.append(ws)
        w = (torch.randn(vocab, HIDDEN, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
        self.lm = (plugin.pack_weight(w), w if keep_bf16 else None)
        self.digit_bytes = sum(2 * N * Kd for _, N, Kd in SHAPES) * layers + 2 * vocab * HIDDEN

    def kv(self, B, L, gen):
        torch = self.torch
        nbp = -(-L // ATT_BS)
        caches = []
        n_att = sum(1 for i in range(len(self.layers)) if i % ATTN_EVERY == ATTN_EVERY - 1)
        for _ in range(n_att):
            kv = torch.randn(B * nbp, ATT_KV, ATT_BS, 2 * ATT_D, device=self.dev, generator=gen,
                             dtype=torch.bfloat16)
            kc, vc = kv.transpose(1, 2).split(ATT_D, dim=-1)
            caches.append((kv, kc, vc))
        bt = torch.randperm(B * nbp, device=self.dev, generator=gen).view(B, nbp).to(torch.int32)
        sl = torch.full((B,), L, device=self.dev, dtype=torch.int32)
        self.max_seq_len = L  # the host bound vLLM's metadata passes with the step
        return caches, bt, sl

    def step(self, h, caches, bt, sl, exact=True):
        torch = self.torch
        B = h.shape[0]

        def lin(x, wp):
            return torch.ops.exactmm.linear(x, *wp[0]) if exact else torch.matmul(x, wp[1].T)

        def rownorm(t):  # t * 2^-e, e = frexp exponent of the row absmax: exact and row-local
            e = torch.frexp(t.abs().amax(dim=-1, keepdim=True).float()).exponent
            return torch.ldexp(t.float(), -e).to(torch.bfloat16)

        a = 0
        for i, ws in enumerate(self.layers):
            qkv = lin(rownorm(h), ws["qkv"])
            if i % ATTN_EVERY == ATTN_EVERY - 1:
                _, kc, vc = caches[a]
                a += 1
                o = torch.empty(B, ATT_H, ATT_D, device=h.device, dtype=torch.bfloat16)
                self.P.paged_decode(qkv[:, :HIDDEN].view(B, ATT_H, ATT_D), kc, vc, bt, sl, ATT_D ** -0.5, o, B,
                                    self.max_seq_len)
                mix = o.view(B, HIDDEN)
            else:
                mix = qkv[:, :HIDDEN]
            h = h + lin(mix, ws["o"])
            gu = lin(rownorm(h), ws["gate_up"])
            half = gu.shape[1] // 2
            h = h + lin(torch.nn.functional.silu(gu[:, :half]) * gu[:, half:], ws["down"])
        return lin(rownorm(h), self.lm)

    def parts(self, B, caches, bt, sl, gen):
        """The three parts of one step, each issued on its own over inputs of the step's shapes,
        for a time breakdown: every linear of the step (the 4 x layers layer linears and the
        lm_head), every attention call, and the glue between them (row rescales, residual adds,
        the gated SiLU). Each callable takes `exact` (False: the hipBLASLt bf16 linears)."""
        torch, dev = self.torch, self.dev
        r = lambda *shape: torch.randn(*shape, device=dev, generator=gen).to(torch.bfloat16)
        xh, xf = r(B, HIDDEN), r(B, FFN)
        gu, q = r(B, 2 * FFN), r(B, ATT_H, ATT_D)
        o = torch.empty(B, ATT_H, ATT_D, device=dev, dtype=torch.bfloat16)

        def linears(exact):
            for ws in self.layers:
                for name, x in (("qkv", xh), ("o", xh), ("gate_up", xh), ("down", xf)):
                    torch.ops.exactmm.linear(x, *ws[name][0]) if exact else torch.matmul(x, ws[name][1].T)
            torch.ops.exactmm.linear(xh, *self.lm[0]) if exact else torch.matmul(xh, self.lm[1].T)

        def attention(exact):
            for _, kc, vc in caches:
                self.P.paged_decode(q, kc, vc, bt, sl, ATT_D ** -0.5, o, B, self.max_seq_len)

        def rownorm(t):
            e = torch.frexp(t.abs().amax(dim=-1, keepdim=True).float()).exponent
            return torch.ldexp(t.float(), -e).to(torch.bfloat16)

        def glue(exact):
            h = xh
            for _ in self.layers:
                rownorm(h)  # before the QKV linear
                h = h + xh  # residual add of the o output
                rownorm(h)  # before gate_up
                torch.nn.functional.silu(gu[:, :FFN]) * gu[:, FFN:]  # the down linear's input
                h = h + xh  # residual add of the down output
            rownorm(h)  # before the lm_head

        return {"linears": linears, "attention": attention, "glue": glue}


def graph_ms(torch, fn, replays=10):
    """Median milliseconds of one replay of a HIP graph holding fn() (captured after a warm
    call on a side stream)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fn()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    ts = []
    for _ in range(replays):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        g.replay()
        e1.record()
        e1.synchronize()
        ts.append(e0.elapsed_time(e1))
    del g
    torch.cuda.synchronize()
    return sorted(ts)[len(ts) // 2]


def gemm_bytes(M, N, K):
    return 2 * N * K + 2 * M * K + 2 * M * N + 8 * N


def gemm_ops(M, N, K, ndots=NDOTS):
    return ndots * 2 * M * N * K


def time_op_and_gemm(torch, K, plugin, x, wc, N, Kd, F, trunc, cfg):
    """Graph-replay times (us) of the full exactmm::linear op on weight copies wc, and of the
    GEMM kernel it runs (the one-launch digitize + GEMM kernel where the table marks the row
    count, else the GEMM on digits made beforehand). Returns (op_us, gemm_us, one_launch)."""
    from vllm_exact.graph_timing import time_graph

    M = x.shape[0]
    nrot = len(wc)
    t_op = time_graph(lambda r: torch.ops.exactmm.linear(x, *wc[r]), nrot)
    out = torch.empty(M, N, device=x.device, dtype=x.dtype)  # the op's output: x's dtype
    one_launch = plugin._one_launch(M, N, Kd)
    if one_launch:
        try:
            K.exact_linear_bf16x(x, (wc[0][0], wc[0][2], wc[0][3]), Kd, F, trunc, out=out, cfg=cfg)
        except NotImplementedError:
            one_launch = False
    if one_launch:
        t_gemm = time_graph(lambda r: K.exact_linear_bf16x(x, (wc[r][0], wc[r][2], wc[r][3]), Kd, F, trunc, out=out,
                                                           cfg=cfg), nrot)
    else:
        xd = K.digitize_packed(x, F)
        t_gemm = time_graph(lambda r: K.exact_linear_packed(xd, (wc[r][0], wc[r][2], wc[r][3]), Kd, F, trunc,
                                                            out=out, cfg=cfg), nrot)
    return t_op, t_gemm, one_launch


def roof_fields(M, N, Kd, t_us, ndots):
    """GB/s, TOPS and roofline fractions of one exact GEMM launch of t_us microseconds."""
    b, o = gemm_bytes(M, N, Kd), gemm_ops(M, N, Kd, ndots)
    t_roof = max(b / (HBM_PEAK_GBS * 1e9), o / (INT8_PEAK_TOPS * 1e12)) * 1e6
    return dict(gemm_GBps=round(b / t_us / 1e3, 1), gemm_TOPS=round(o / t_us / 1e6, 1),
                hbm_frac=round(b / t_us / 1e3 / HBM_PEAK_GBS, 3), mfma_frac=round(o / t_us / 1e6 / INT8_PEAK_TOPS, 3),
                roofline_frac=round(t_roof / t_us, 3),
                bound="hbm" if b / (HBM_PEAK_GBS * 1e9) >= o / (INT8_PEAK_TOPS * 1e12) else "mfma")


def sampled_rows_exact(torch, np, oracle, x, wd, y, Fx, trunc):
    """True when the bf16 output rows 0..7, M/2 and M-1 of y = exactmm::linear(x, w) equal,
    bit for bit, the oracle's result on the same rows (wd: the oracle's digits of w at Fx)."""
    M = x.shape[0]
    rows = np.unique(np.concatenate([np.arange(min(M, 8)), [M // 2, M - 1]]))
    ref = oracle.exact_linear_c(oracle.digitize_c(x.float().cpu().numpy()[rows], Fx), wd, Fx, trunc)
    got = y[rows.tolist()].cpu().view(torch.int16).numpy().view(np.uint16)
    return bool(np.array_equal(got, oracle.bf16_rne_c(ref).reshape(ref.shape)))


def sweep_f15(torch, K, plugin, weights, xs, table_f15, table_f14, np, oracle):
    """The 4-dot variant: the sweep at F = 15 (offset digits, the reference's "f=15, 4 dots")
    with the table tuned at F = 15, each op through exactmm::linear on weights packed at
    F = 15, timed like the F = 14 sweep and its sampled output rows checked bitwise against
    the oracle. Restores F = 14 and its table afterwards."""
    from vllm_exact.graph_timing import rotations_for

    recs = []
    plugin.F, plugin.TRUNC = 15, False
    plugin.load_table(table_f15)
    try:
        for name, N, Kd in SHAPES:
            w = weights[name + ".bf16"]
            wp = plugin.pack_weight(w)
            wc = [wp] + [tuple(t.clone() for t in wp) for _ in range(max(3, rotations_for(2 * N * Kd)) - 1)]
            wd = oracle.digitize_c(w.float().cpu().numpy(), 15)
            for M in MS:
                cfg = plugin._cfg(M, N, Kd)
                t_op, t_gemm, one = time_op_and_gemm(torch, K, plugin, xs[(M, Kd)], wc, N, Kd, 15, False, cfg)
                exact = sampled_rows_exact(torch, np, oracle, xs[(M, Kd)], wd,
                                           torch.ops.exactmm.linear(xs[(M, Kd)], *wc[0]), 15, False)
                rec = dict(M=M, op=name, N=N, K=Kd, cfg=list(cfg), op_us=round(t_op, 2), gemm_us=round(t_gemm, 2),
                           one_launch=one, bit_exact=exact, **roof_fields(M, N, Kd, t_gemm, 4))
                recs.append(rec)
                log("f15", json.dumps(rec))
            del wc, wp
            torch.cuda.empty_cache()
    finally:
        plugin.F, plugin.TRUNC = F, TRUNC
        plugin.load_table(table_f14)
    return recs


def config1(torch, K, plugin, oracle, np, dev, gen):
    """The reference's CPU-runnable case on the GPU: M = 16, K = N = 4096, F = 14 with all four
    dots, no split-K (the F = 14 table's cfg for the shape with SK = 1). The GEMM kernel and the
    full op (digitize + GEMM) timed by graph replay over weight copies past the MALL; the whole
    fp32 and bf16 outputs checked bitwise against the oracle."""
    from vllm_exact.graph_timing import rotations_for, time_graph

    M, N, Kd, Fc, trunc = 16, 4096, 4096, 14, False
    cfg = tuple(plugin._cfg(M, N, Kd)[:6]) + (1,)
    x = torch.randn(M, Kd, device=dev, generator=gen).to(torch.bfloat16)
    w = (torch.randn(N, Kd, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
    wp = K.digitize_packed(w, Fc)
    wc = [wp] + [tuple(t.clone() for t in wp) for _ in range(rotations_for(2 * N * Kd) - 1)]
    xd = K.digitize_packed(x, Fc)
    ob = torch.empty(M, N, device=dev, dtype=torch.bfloat16)  # timed with the op's bf16 output
    t_gemm = time_graph(lambda r: K.exact_linear_packed(xd, wc[r], Kd, Fc, trunc, out=ob, cfg=cfg), len(wc))
    t_two = time_graph(lambda r: K.exact_linear_packed(K.digitize_packed(x, Fc), wc[r], Kd, Fc, trunc, out=ob,
                                                       cfg=cfg), len(wc))
    try:
        t_one = time_graph(lambda r: K.exact_linear_bf16x(x, wc[r], Kd, Fc, trunc, out=ob, cfg=cfg), len(wc))
    except NotImplementedError:
        t_one = None
    y32 = K.exact_linear_packed(xd, wp, Kd, Fc, trunc, cfg=cfg).cpu().numpy()
    yb = K.exact_linear_packed(xd, wp, Kd, Fc, trunc, cfg=cfg, out=torch.empty(M, N, device=dev,
                                                                                dtype=torch.bfloat16))
    ref = oracle.exact_linear_c(oracle.digitize_c(x.float().cpu().numpy(), Fc),
                                oracle.digitize_c(w.float().cpu().numpy(), Fc), Fc, trunc)
    exact = bool(np.array_equal(y32.view(np.uint32), ref.view(np.uint32))) and bool(np.array_equal(
        yb.cpu().view(torch.int16).numpy().view(np.uint16), oracle.bf16_rne_c(ref).reshape(M, N)))
    t_op = min(t for t in (t_two, t_one) if t is not None)
    rec = dict(M=M, N=N, K=Kd, F=Fc, trunc=trunc, ndots=4, cfg=list(cfg), gemm_us=round(t_gemm, 2),
               op_us=round(t_op, 2), op_two_launch_us=round(t_two, 2),
               op_one_launch_us=None if t_one is None else round(t_one, 2), bit_exact_fp32_bf16=exact,
               **roof_fields(M, N, Kd, t_gemm, 4))
    log("config 1:", json.dumps(rec))
    return rec


def cpu_baseline_leg(torch, K, np, oracle, step_bytes, ops, budget_s):
    """The reference's CPU path timed on this host: digitize_torch + exact_linear_torch, the
    torch int64 statements of kernels.py:22-39, 89-100, on every host thread. Config 1
    (16 x 4096 x 4096, 4 dots) runs in full; each sweep op runs on a sample of its weight rows
    (rows are independent), its time extrapolated linearly in N (the activation digitize is
    timed once, unscaled). Weights are digitized beforehand, as the reference does at load.
    The C oracle (OpenMP) is timed beside it on the same sample budget."""
    ncpu = os.cpu_count()
    torch.set_num_threads(ncpu)
    threads = torch.get_num_threads()
    g = torch.Generator().manual_seed(0)

    def timed(fn, min_s):
        reps, t0 = 0, time.perf_counter()
        while True:
            fn()
            reps += 1
            dt = (time.perf_counter() - t0) / reps
            if reps * dt >= min_s or reps >= 1000:
                return dt, reps

    # config 1 in full
    x1 = torch.randn(16, 4096, generator=g).to(torch.bfloat16).float()
    w1 = (torch.randn(4096, 4096, generator=g) * 0.02).to(torch.bfloat16).float()
    wd1 = K.digitize_torch(w1, 14)
    t1, r1 = timed(lambda: K.exact_linear_torch(K.digitize_torch(x1, 14), wd1, 14, trunc=False), 1.0)
    c1 = dict(seconds=round(t1, 4), GBps=round(gemm_bytes(16, 4096, 4096) / t1 / 1e9, 3),
              GOPs=round(gemm_ops(16, 4096, 4096, 4) / t1 / 1e9, 3), reps=r1, sample="full (not extrapolated)")

    # the sweep: sampled weight rows per op
    per_op_s = budget_s / len(ops)
    # at most 2048 weight rows a shape are sampled
    wfull = {name: (torch.randn(min(N, 2048), Kd, generator=g) * 0.02).to(torch.bfloat16).float()
             for name, N, Kd in SHAPES}
    total_s, desc, op_s = 0.0, [], {}
    for M, name, N, Kd in ops:
        x = torch.randn(M, Kd, generator=g).to(torch.bfloat16).float()
        t_dig, _ = timed(lambda: K.digitize_torch(x, F), 0.05)
        xd = K.digitize_torch(x, F)
        # calibrate on 64 weight rows, then a sample sized so that about three repetitions fill
        # the op's share of the budget; the time is the mean over the repetitions timed
        wd = K.digitize_torch(wfull[name][:64], F)
        t0 = time.perf_counter()
        K.exact_linear_torch(xd, wd, F, TRUNC)
        per_row = (time.perf_counter() - t0) / 64
        ns = int(min(N, 2048, max(64, per_op_s / 3 / max(per_row, 1e-9)))) // 16 * 16
        wd = K.digitize_torch(wfull[name][:ns], F)
        t_lin, reps = timed(lambda: K.exact_linear_torch(xd, wd, F, TRUNC), per_op_s * 2 / 3)
        t = t_dig + t_lin * N / ns
        op_s[(M, name)] = t
        total_s += t
        desc.append(f"M={M} {name} {ns}/{N} rows x{reps}")
    cpu = dict(value=round(step_bytes / total_s / 1e9, 4), unit="GB/s", cores=threads, kind="port",
               os_cpu_count=ncpu, torch_threads=threads,
               sample="torch int64 statements of the reference's CPU path (kernels.digitize_torch + "
                      "kernels.exact_linear_torch) on every host thread; each sweep op on its first weight rows, "
                      "mean over the repetitions shown (xN), time extrapolated linearly in N (labelled "
                      "extrapolated); config 1 in full: "
                      + "; ".join(desc),
               step_ms_extrapolated=round(total_s * 1e3, 1), config1_full=c1)

    # the C oracle on the same kind of sample
    rng = np.random.default_rng(0)
    samples = {}
    for name, N, Kd in SHAPES:
        ns = min(N, 2048)
        samples[name] = (ns, oracle.digitize_c((rng.standard_normal((ns, Kd)) * 0.02).astype(np.float32), F))
    oc_total, oc_desc, oc_op = 0.0, [], {}
    for M, name, N, Kd in ops:
        ns, wd = samples[name]
        x = rng.standard_normal((M, Kd)).astype(np.float32)
        dt, reps = timed(lambda: oracle.exact_linear_c(oracle.digitize_c(x, F), wd, F, TRUNC), per_op_s / 3)
        oc_op[(M, name)] = dt * N / ns
        oc_total += dt * N / ns
        oc_desc.append(f"M={M} {name} {ns}/{N} rows x{reps}")
    cpu["oracle_c"] = dict(value=round(step_bytes / oc_total / 1e9, 3), unit="GB/s", cores=oracle.cpu_threads(),
                           step_ms_extrapolated=round(oc_total * 1e3, 1),
                           sample="C oracle (digitize + exact integer digit dots, OpenMP), time extrapolated "
                                  "linearly in N: " + "; ".join(oc_desc))
    log("cpu baseline:", json.dumps(cpu))
    return cpu, op_s


def parse():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--no-attention", action="store_true")
    ap.add_argument("--no-cpu", action="store_true")
    ap.add_argument("--no-decode-step", action="store_true")
    ap.add_argument("--no-lm-head", action="store_true")
    ap.add_argument("--cpu-seconds", type=float, default=15.0, help="target CPU-baseline sample time")
    ap.add_argument("--table", default=str(ROOT / "vllm-exact_amd" / "vllm_exact" / "cfg_table_mi355x_F14.json"),
                    help="exact_int8 tuning table to use")
    ap.add_argument("--table-f15", default=str(ROOT / "vllm-exact_amd" / "vllm_exact" / "cfg_table_mi355x_F15.json"),
                    help="tuning table of the 4-dot F = 15 sweep (per_op_f15)")
    ap.add_argument("--no-f15", action="store_true", help="skip the 4-dot F = 15 sweep and the config-1 timing")
    ap.add_argument("--profile-counters", action="store_true",
                    help="only launch every sweep GEMM (table cfg, weights rotated past the MALL) and the three "
                         "decode-attention shapes, 5 times each, then a 1 GiB copy: the program rocprofv3 --pmc "
                         "passes (MFMA utilisation, FETCH_SIZE, WRITE_SIZE) run; one JSON line per launch group")
    ap.add_argument("--floors", action="store_true",
                    help="only measure the achievable ceilings of the paths the kernels run on (vllm-exact_amd/floors): "
                         "MFMA issue rate, LDS read rate, L2-resident load rate into VGPRs and straight into LDS, "
                         "streaming reads at the sweep's weight sizes (graph replay, buffers rotated past the MALL) "
                         "and reads of permuted 8 KiB pages; one JSON line")
    ap.add_argument("--profile-kernel", action="store_true",
                    help="only launch the dominant GEMM (M=256 gate_up, table cfg) and a 1 GiB copy, --steps times "
                         "each: the program rocprofv3 --pmc FETCH_SIZE / WRITE_SIZE runs to measure HBM traffic")
    return ap.parse_args()


TRAFFIC_SUMMARY = ROOT / "profiles" / "exact_gemm_m256_gate_up_hbm_traffic.md"
COUNTERS_SUMMARY = ROOT / "profiles" / "exact_gemm_and_attention_counters.md"


# The library's sources that no linear is built from: attention, the 8-bit cache and their calls.
OTHER_SOURCES = {"attention_common.h", "beam_select.hip", "int8_cache.hip", "linear_attention.hip", "paged_decode.hip", "pages.hip",
                 "prompt_attention.hip", "tensor_calls.cpp", "tree_decode.hip"}


def kernel_sources():
    """The csrc/ files that the linears' kernels are built from."""
    files = (ROOT / "vllm-exact_amd" / "csrc").glob("*")
    return sorted(f for f in files if f.is_file() and f.name not in OTHER_SOURCES)


def kernel_sources_sha16():
    """Hash of the sources that the linears' kernels are built from: a traffic figure measured on
    one build is only reported for a library whose linears are built from the same sources. Another
    operator beside them changes nothing here."""
    import hashlib

    h = hashlib.sha256()
    for f in kernel_sources():
        h.update(f.name.encode() + b"\0" + f.read_bytes())
    return h.hexdigest()[:16]


def read_traffic(kernel_cfg):
    """HBM bytes per launch of the dominant GEMM, as measured by the rocprofv3 FETCH_SIZE and
    WRITE_SIZE passes of `bench.py --profile-kernel` and recorded in TRAFFIC_SUMMARY (its
    `traffic_bytes_per_launch`, `cfg` and `kernel_sources_sha16` lines). Returns (bytes,
    where the figure comes from), or (None, why not) when the summary was measured with
    another cfg or on a library built from other sources."""
    if not TRAFFIC_SUMMARY.exists():
        return None, "no traffic summary"
    vals = {}
    for line in TRAFFIC_SUMMARY.read_text().splitlines():
        if line.startswith("    ") and "=" in line:
            k, v = line.strip().split("=", 1)
            vals[k.strip()] = v.strip()
    try:
        if json.loads(vals["cfg"]) != list(kernel_cfg):
            return None, f"{TRAFFIC_SUMMARY.name} was measured with cfg {vals['cfg']}"
        if vals.get("kernel_sources_sha16") != kernel_sources_sha16():
            return None, f"{TRAFFIC_SUMMARY.name} was measured on a library built from other sources"
        return int(vals["traffic_bytes_per_launch"]), (
            f"profiles/{TRAFFIC_SUMMARY.name}: rocprofv3 FETCH_SIZE + WRITE_SIZE of bench.py --profile-kernel on "
            f"this library's sources (sha16 {vals['kernel_sources_sha16']}), calibrated on a 1 GiB copy")
    except (KeyError, ValueError):
        return None, f"{TRAFFIC_SUMMARY.name} is incomplete"


def read_op_traffic():
    """Per sweep op, the HBM bytes per launch (GEMM + split-K finalize) measured by the
    FETCH_SIZE and WRITE_SIZE passes of `bench.py --profile-counters`, as recorded in
    COUNTERS_SUMMARY: its `kernel_sources_sha16` line and one `traffic M:<M> op:<op> cfg:<cfg>
    = <bytes>` line per op. Returns ({(M, op): (bytes, cfg)}, note); empty when the record was
    made on a library built from other sources."""
    if not COUNTERS_SUMMARY.exists():
        return {}, "no counters summary"
    out, sha = {}, None
    for line in COUNTERS_SUMMARY.read_text().splitlines():
        if not line.startswith("    ") or "=" not in line:
            continue
        k, v = line.strip().rsplit("=", 1)
        k, v = k.strip(), v.strip()
        if k == "kernel_sources_sha16":
            sha = v
        elif k.startswith("traffic "):
            f = dict(t.split(":", 1) for t in k.split()[1:])
            out[(int(f["M"]), f["op"])] = (int(v), json.loads(f["cfg"]))
    if sha != kernel_sources_sha16():
        return {}, f"{COUNTERS_SUMMARY.name} was measured on a library built from other sources"
    return out, f"profiles/{COUNTERS_SUMMARY.name} (sha16 {sha})"


def profile_kernel(args):
    """Launch the dominant GEMM --steps times, its weights rotated over copies as in the timed
    run, then a plain copy of known size --steps times (kernel-trace and counter runs)."""
    import torch

    from vllm_exact import _native
    from vllm_exact import kernels as K
    from vllm_exact import plugin
    from vllm_exact.graph_timing import rotations_for

    _native.lib()
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    plugin.load_table(args.table)
    gen = torch.Generator(device=dev).manual_seed(0)
    M, (name, N, Kd) = 256, SHAPES[2]
    cfg = plugin._cfg(M, N, Kd)
    w = (torch.randn(N, Kd, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
    wp, _, cw, sw = plugin.pack_weight(w)
    rot = rotations_for(2 * N * Kd)
    wps = [wp] + [wp.clone() for _ in range(rot - 1)]
    x = torch.randn(M, Kd, device=dev, generator=gen).to(torch.bfloat16)
    xd = K.digitize_packed(x, F)
    out = torch.empty(M, N, device=dev, dtype=torch.bfloat16)
    src = torch.randn(1 << 29, device=dev, generator=gen).to(torch.bfloat16)  # 1 GiB
    dst = torch.empty_like(src)
    torch.cuda.synchronize()
    for i in range(args.steps):
        K.exact_linear_packed(xd, (wps[i % rot], cw, sw), Kd, F, TRUNC, out=out, cfg=cfg)
    torch.cuda.synchronize()
    for _ in range(args.steps):
        dst.copy_(src)
    torch.cuda.synchronize()
    print(json.dumps({"gemm": f"M={M} {name} {N}x{Kd}", "cfg": list(cfg), "launches": args.steps,
                      "weight_copies": rot, "copy_bytes": src.numel() * 2,
                      "algorithmic_bytes": gemm_bytes(M, N, Kd), "kernel_sources_sha16": kernel_sources_sha16()}),
          flush=True)


def profile_counters(args):
    """Launch each sweep GEMM and each decode-attention shape a few times, in a fixed order, for
    rocprofv3 counter passes; print one JSON line per group (what ran, how many launches, its
    algorithmic bytes and ops) so the counter rows can be matched to the ops."""
    import torch

    from vllm_exact import _native
    from vllm_exact import kernels as K
    from vllm_exact import paged_attn as P
    from vllm_exact import plugin
    from vllm_exact.graph_timing import rotations_for

    _native.lib()
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    plugin.load_table(args.table)
    gen = torch.Generator(device=dev).manual_seed(0)
    print(json.dumps({"group": "meta", "kernel_sources_sha16": kernel_sources_sha16()}), flush=True)
    n = 5
    for name, N, Kd in SHAPES:
        w = (torch.randn(N, Kd, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
        w0 = plugin.pack_weight(w)
        wc = [w0] + [tuple(t.clone() for t in w0) for _ in range(rotations_for(2 * N * Kd) - 1)]
        for M in MS:
            cfg = plugin._cfg(M, N, Kd)
            x = torch.randn(M, Kd, device=dev, generator=gen).to(torch.bfloat16)
            xd = K.digitize_packed(x, F)
            out = torch.empty(M, N, device=dev, dtype=torch.bfloat16)
            torch.cuda.synchronize()
            for i in range(n):
                r = wc[i % len(wc)]
                K.exact_linear_packed(xd, (r[0], r[2], r[3]), Kd, F, TRUNC, out=out, cfg=cfg)
            torch.cuda.synchronize()
            print(json.dumps({"group": "gemm", "op": name, "M": M, "N": N, "K": Kd, "cfg": list(cfg), "launches": n,
                              "algorithmic_bytes": gemm_bytes(M, N, Kd), "algorithmic_ops": gemm_ops(M, N, Kd)}),
                  flush=True)
        del wc, w0
        torch.cuda.empty_cache()
    H, KV, D, BS = 32, 8, 128, 16
    P.MAX_LEN = 16384
    for B, L in ATTN_CASES:
        nbp = L // BS
        kv = torch.randn(B * nbp, KV, BS, 2 * D, device=dev, generator=gen, dtype=torch.bfloat16)
        bt = torch.randperm(B * nbp, device=dev, generator=gen).view(B, nbp).to(torch.int32)
        q = torch.randn(B, H, D, device=dev, generator=gen, dtype=torch.bfloat16)
        sl = torch.full((B,), L, device=dev, dtype=torch.int32)
        kc, vc = kv.transpose(1, 2).split(D, dim=-1)
        out = torch.empty(B, H, D, device=dev, dtype=torch.bfloat16)
        torch.cuda.synchronize()
        for _ in range(3):
            P.paged_decode(q, kc, vc, bt, sl, D ** -0.5, out, B, L)
        torch.cuda.synchronize()
        print(json.dumps({"group": "attention", "B": B, "L": L, "launches": 3, "kv_bytes": B * L * KV * D * 2 * 2}),
              flush=True)
        del kv, kc, vc
        torch.cuda.empty_cache()
    src = torch.randn(1 << 29, device=dev, generator=gen).to(torch.bfloat16)  # 1 GiB
    dst = torch.empty_like(src)
    torch.cuda.synchronize()
    for _ in range(3):
        dst.copy_(src)
    torch.cuda.synchronize()
    print(json.dumps({"group": "copy", "launches": 3, "bytes": src.numel() * 2}), flush=True)

FLOORS_LIB = ROOT / "vllm-exact_amd" / "vllm_exact" / "libvxa_floors.so"
FLOORS_SRC = ROOT / "vllm-exact_amd" / "floors" / "floors.hip"


def floors(args):
    """Achievable ceilings of the paths the exact GEMM and the attention run on, measured with
    the probe kernels of vllm-exact_amd/floors/floors.hip (which compute nothing useful). Each
    kernel-timed figure is one launch timed with HIP events on torch's stream; the streaming
    reads at the sweep's weight sizes are timed like the GEMMs (graph replay, buffers rotated
    past the MALL). Each probe's shader clock is its workgroups' s_memtime cycles over their
    s_memrealtime ticks (100 MHz)."""
    import ctypes
    import hashlib
    import statistics

    import torch

    from vllm_exact.graph_timing import rotations_for, time_graph

    lib = ctypes.CDLL(str(FLOORS_LIB))
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    lib.vxf_stream.argtypes = [vp, i64, i64, i32, i32, i32, i32, vp, vp, vp]
    lib.vxf_pages.argtypes = [vp, i64, vp, i32, i32, i32, i32, vp, vp, vp]
    lib.vxf_wave_pages.argtypes = [vp, i64, vp, i32, i32, i32, i32, vp, vp, vp]
    lib.vxf_l2.argtypes = [vp, i64, i32, i32, i32, i32, i32, vp, vp, vp]
    lib.vxf_lds.argtypes = [i32, i32, i32, vp, vp, vp]
    lib.vxf_mfma.argtypes = [i32, i32, i32, vp, vp, vp]
    lib.vxf_mfma_shape.argtypes = [i32, i32, i32, i32, vp, vp, vp]
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    ncu = torch.cuda.get_device_properties(dev).multi_processor_count
    max_blocks = 4096
    sink = torch.zeros(max_blocks * 1024, device=dev, dtype=torch.int32)
    cyc = torch.zeros(2 * max_blocks, device=dev, dtype=torch.int64)  # shader cycles, then 100 MHz ticks

    def st():
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def check(rc):
        if rc != 0:
            raise RuntimeError(f"floors probe refused its arguments or failed to launch (status {rc})")

    def timed(launch, blocks, reps=5):
        """Median event time (us) of one launch, the mean shader cycles of its workgroups, and the
        shader clock (GHz) they ran at: their s_memtime cycles over their s_memrealtime ticks."""
        assert blocks <= max_blocks
        launch()
        torch.cuda.synchronize()
        us, cycles, ghz = [], [], []
        for _ in range(reps):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            launch()
            b.record()
            b.synchronize()
            us.append(a.elapsed_time(b) * 1000.0)
            c = cyc[:2 * blocks].double().view(2, blocks)
            cycles.append(c[0].mean().item())
            ghz.append(c[0].sum().item() / c[1].sum().item() * 0.1)
        return statistics.median(us), statistics.median(cycles), statistics.median(ghz)

    out = {"mode": "floors", "cus": ncu, "source_sha16": hashlib.sha256(FLOORS_SRC.read_bytes()).hexdigest()[:16]}

    # MFMA issue rate: 8 independent v_mfma_i32_16x16x64_i8 chains per wave, one workgroup per CU
    mf = []
    for waves in (4, 8, 16):
        rounds = 4096
        us, _, ghz_run = timed(lambda: check(lib.vxf_mfma(waves, ncu, rounds, sink.data_ptr(), cyc.data_ptr(), st())),
                               ncu)
        per_simd = rounds * 8 * waves / 4
        ops = ncu * waves * rounds * 8 * 16 * 16 * 64 * 2
        mf.append({"waves_per_cu": waves, "us": round(us, 1), "ghz": round(ghz_run, 3),
                   "cycles_per_mfma_per_simd": round(us * 1e3 * ghz_run / per_simd, 2), "TOPS": round(ops / us / 1e6, 1)})
        log("mfma", mf[-1])
    out["mfma_i8_16x16x64"] = mf
    ghz = mf[0]["ghz"]

    # The two INT8 MFMA shapes at equal work, 8 waves per CU: operands the same in every
    # instruction, or random with a different set in every instruction (the power a GEMM's
    # digit fragments draw sets the clock)
    ms = []
    for shape in (16, 32):
        for rnd in (0, 1):
            rounds = 8192
            us, _, ghz_run = timed(lambda: check(lib.vxf_mfma_shape(shape, rnd, ncu, rounds, sink.data_ptr(),
                                                                    cyc.data_ptr(), st())), ncu)
            ops = ncu * 8 * rounds * 8 * 16 * 16 * 64 * 2
            peak_per_ghz = ncu * 4 * 2048 * 1e9  # INT8 ops per second per GHz: 2048 per clock per SIMD
            ms.append({"shape": f"{shape}x{shape}x{1024 // shape}", "operands": "random" if rnd else "constant",
                       "us": round(us, 1), "ghz": round(ghz_run, 3), "TOPS": round(ops / us / 1e6, 1),
                       "frac_of_peak_at_clock": round(ops / (us * 1e-6) / (peak_per_ghz * ghz_run), 3)})
            log("mfma_shape", ms[-1])
    out["mfma_i8_shapes"] = ms

    # LDS reads: ds_read_b128, 8 in flight per lane
    ld = []
    for waves in (4, 8, 16):
        rounds = 2048
        us, _, ghz_run = timed(lambda: check(lib.vxf_lds(waves, ncu, rounds, sink.data_ptr(), cyc.data_ptr(), st())),
                               ncu)
        b = rounds * 8 * 64 * 16 * waves
        ld.append({"waves_per_cu": waves, "us": round(us, 1), "ghz": round(ghz_run, 3),
                   "bytes_per_clk_per_cu": round(b / (us * 1e3 * ghz_run), 1)})
        log("lds", ld[-1])
    out["lds_read_b128"] = ld

    # L2-resident loads (2 MiB buffer: every XCD's L2 holds it), into VGPRs or straight into LDS
    l2buf = torch.zeros(1 << 21, device=dev, dtype=torch.uint8)
    l2 = []
    for lds in (0, 1):
        for waves in (4, 8, 16):
            for q in (1, 2, 4, 8):
                rounds = max(64, 16384 // (q * waves))
                us, _, ghz_run = timed(lambda: check(lib.vxf_l2(l2buf.data_ptr(), l2buf.numel(), lds, q, waves, ncu,
                                                                rounds, sink.data_ptr(), cyc.data_ptr(), st())), ncu)
                b = rounds * q * 1024 * waves
                l2.append({"path": "lds" if lds else "vgpr", "waves_per_cu": waves, "loads_in_flight": q,
                           "us": round(us, 1), "ghz": round(ghz_run, 3),
                           "bytes_per_clk_per_cu": round(b / (us * 1e3 * ghz_run), 1),
                           "TBps": round(b * ncu / us / 1e6, 2)})
                log("l2", l2[-1])
    out["l2_load_16B"] = l2

    # The shader clock under the large-M GEMM's mix: MFMAs with loads in about its proportion (56
    # MFMAs per 8 KiB a wave loads: 146 bytes per MFMA per CU, where the M = 256 gate_up tile loads
    # 2.62 MB per 18,432 MFMAs), the loads all L2-resident or a quarter of them streamed from HBM
    # (a 1 GiB buffer, past the MALL), and under each part alone; the MFMA operands constant or
    # redrawn every round (random bits, as the GEMM's digits). Three launches of about 1-2 ms back
    # to back; the clock of the last, per workgroup, from s_memtime over s_memrealtime.
    lib.vxf_mfma_mix.argtypes = [vp, i64, vp, i64, i32, i32, i32, i32, i32, vp, vp, vp]
    clk = torch.zeros(2 * ncu, device=dev, dtype=torch.int64)
    hbuf = torch.empty(1 << 30, device=dev, dtype=torch.uint8)
    under = []
    for loads, mfmas, vary in ((1, 0, 0), (2, 0, 0), (0, 56, 0), (0, 56, 1), (1, 56, 0), (1, 56, 1), (2, 56, 0),
                               (2, 56, 1)):
        rounds = 2000

        def launch(loads=loads, mfmas=mfmas, vary=vary):
            check(lib.vxf_mfma_mix(l2buf.data_ptr(), l2buf.numel(), hbuf.data_ptr(), hbuf.numel(), loads, mfmas, vary,
                                   ncu, rounds, sink.data_ptr(), clk.data_ptr(), st()))

        launch()
        torch.cuda.synchronize()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(3):
            launch()
        b.record()
        b.synchronize()
        us = a.elapsed_time(b) * 1000.0 / 3
        c = clk.view(-1, 2).double()
        ghz_wg = (c[:, 0] / c[:, 1] * 0.1).cpu()
        cycles = float(c[:, 0].median())
        row = {"loads": ["none", "l2", "l2_and_hbm"][loads], "mfmas_per_8KiB": mfmas,
               "mfma_operands": "random" if vary else "constant", "us": round(us, 1),
               "ghz_median": round(float(ghz_wg.median()), 3), "ghz_min": round(float(ghz_wg.min()), 3),
               "ghz_max": round(float(ghz_wg.max()), 3)}
        if loads:
            row["bytes_per_clk_per_cu"] = round(rounds * 8 * 8192 / cycles, 1)
            if loads == 2:
                row["hbm_TBps"] = round(ncu * rounds * 2 * 8192 / us / 1e6, 2)
        if mfmas:
            row["TOPS"] = round(ncu * 8 * rounds * mfmas * 16 * 16 * 64 * 2 / us / 1e6, 1)
        under.append(row)
        log("clock under load", row)
    del hbuf
    out["clock_under_gemm_mix"] = under
    del l2buf

    # Streaming reads at the sweep's weight sizes, timed like the GEMMs, with nontemporal loads
    # (what the GEMMs use for weights read once) and with the default cache policy
    sizes = {"o": 4096 * 4096 * 2, "qkv": 6144 * 4096 * 2, "down": 4096 * 12288 * 2, "gate_up": 24576 * 4096 * 2}
    stream_rows = []
    for name, nbytes in sizes.items():
        rot = rotations_for(nbytes)
        bufs = [torch.empty(nbytes, device=dev, dtype=torch.uint8) for _ in range(rot)]
        for nt in (1, 0):
            best = None
            for blocks in (256, 512, 1024):
                for q in (4, 8):
                    per_wg = nbytes // blocks
                    per_wg -= per_wg % (16 * 512)
                    if per_wg <= 0:
                        continue

                    def call(i, blocks=blocks, q=q, per_wg=per_wg, nt=nt):
                        check(lib.vxf_stream(bufs[i].data_ptr(), nbytes, per_wg, blocks, 512, q, nt, sink.data_ptr(),
                                             cyc.data_ptr(), st()))

                    us = time_graph(call, rotations=rot)
                    row = {"blocks": blocks, "loads_in_flight": q, "us": round(us, 2), "bytes_read": per_wg * blocks,
                           "hbm_frac": round(per_wg * blocks / us / 1e3 / HBM_PEAK_GBS, 3)}
                    if best is None or row["us"] < best["us"]:
                        best = row
            stream_rows.append({"weights_of": name, "bytes": nbytes, "copies": rot,
                                "policy": "nontemporal" if nt else "default", **best})
            log("stream", stream_rows[-1])
        del bufs
        torch.cuda.empty_cache()
    empty_us = time_graph(lambda i: check(lib.vxf_mfma(4, 1, 1, sink.data_ptr(), cyc.data_ptr(), st())))
    out["stream_read"] = stream_rows
    out["empty_launch_us"] = round(empty_us, 2)

    # The packed digitize (the op's first launch) against a copy with its grid and traffic and no
    # arithmetic, graph replay with the launch included, inputs rotated over four copies
    from vllm_exact import kernels as K
    lib.vxf_rowcopy.argtypes = [vp, i64, i64, i64, vp, i64, vp]
    dg = []
    for rows, k in ((64, 4096), (256, 4096), (256, 12288)):
        xs = [torch.randn(rows, k, device=dev).to(torch.bfloat16) for _ in range(4)]
        hbuf = torch.empty(rows * k * 2, device=dev, dtype=torch.int8)
        t_dig = statistics.median(time_graph(lambda i: K.digitize_packed(xs[i], 14), 4) for _ in range(3))
        t_copy = statistics.median(
            time_graph(lambda i: check(lib.vxf_rowcopy(xs[i].data_ptr(), xs[i].numel() * 2, rows, k, hbuf.data_ptr(),
                                                       hbuf.numel(), st())), 4) for _ in range(3))
        dg.append({"rows": rows, "K": k, "digitize_us": round(t_dig, 2), "rowcopy_us": round(t_copy, 2)})
        log("digitize", dg[-1])
        del xs, hbuf
    out["digitize_vs_rowcopy"] = dg

    # Permuted 8 KiB pages (the paged KV stream): 1 GiB, each page read once
    nb = 1 << 30
    pbuf = torch.empty(nb, device=dev, dtype=torch.uint8)
    npg = nb // 8192
    gen = torch.Generator(device=dev).manual_seed(0)
    perm = torch.randperm(npg, device=dev, generator=gen).to(torch.int32)
    assert int(perm.max()) < npg and int(perm.min()) >= 0
    pg = []
    for nt in (1, 0):
        for blocks in (1024, 2048, 4096):
            ppw = npg // blocks
            for q in (1, 2, 4):
                us, _, _ = timed(lambda: check(lib.vxf_pages(pbuf.data_ptr(), nb, perm.data_ptr(), blocks, ppw, q, nt,
                                                          sink.data_ptr(), cyc.data_ptr(), st())), blocks)
                pg.append({"policy": "nontemporal" if nt else "default", "blocks": blocks, "pages_in_flight": q,
                           "us": round(us, 1), "TBps": round(blocks * ppw * 8192 / us / 1e6, 2)})
                log("pages", pg[-1])
    out["permuted_8k_pages"] = pg
    # one wave per page in the attention kernel's lane pattern, 4 workgroups of 4 waves per CU
    # (36 KiB of LDS each), as the attention kernel runs at 4 waves per SIMD
    wp = []
    for nt in (1, 0):
        for blocks in (1024, 2048):
            ppw = npg // (blocks * 4)
            assert blocks * 4 * ppw <= npg
            us, _, _ = timed(lambda: check(lib.vxf_wave_pages(pbuf.data_ptr(), nb, perm.data_ptr(), blocks, ppw, nt,
                                                           36 * 1024, sink.data_ptr(), cyc.data_ptr(), st())), blocks)
            wp.append({"policy": "nontemporal" if nt else "default", "blocks": blocks, "us": round(us, 1),
                       "TBps": round(blocks * 4 * ppw * 8192 / us / 1e6, 2)})
            log("wave_pages", wp[-1])
    out["permuted_8k_pages_one_wave_each_attention_lanes"] = wp
    seq = torch.arange(npg, device=dev, dtype=torch.int32)
    us, _, _ = timed(lambda: check(lib.vxf_pages(pbuf.data_ptr(), nb, seq.data_ptr(), 2048, npg // 2048, 2, 1,
                                              sink.data_ptr(), cyc.data_ptr(), st())), 2048)
    out["sequential_8k_pages_TBps"] = round(nb / us / 1e6, 2)
    out["ghz_one_wave_per_simd_mfma"] = ghz
    print(json.dumps(out), flush=True)



def log(*a):
    print(*a, file=sys.stderr, flush=True)


def main():
    args = parse()
    if args.gpus != 1 or int(os.environ.get("WORLD_SIZE", "1")) != 1:
        print(json.dumps({"error": "this build measures one GPU only: the exact linear path is a per-GPU kernel "
                                   "library (multi-GPU sharding is a design note); run with --gpus 1"}))
        sys.exit(2)
    if args.profile_kernel:
        profile_kernel(args)
        return
    if args.profile_counters:
        profile_counters(args)
        return
    if args.floors:
        floors(args)
        return
    import numpy as np
    import torch

    from vllm_exact import _native
    from vllm_exact import kernels as K
    from vllm_exact import paged_attn as P
    from vllm_exact import plugin
    from vllm_exact.graph_timing import rotations_for, time_graph

    _native.lib()
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    plugin.load_table(args.table)
    plugin.F, plugin.TRUNC = F, TRUNC
    gen = torch.Generator(device=dev).manual_seed(0)

    # ---------------------------------------------------------------- weights and inputs
    total_w = sum(2 * N * Kd for _, N, Kd in SHAPES)
    rot = rotations_for(total_w, min_total=3 * total_w, min_rot=3)
    weights = {}
    for name, N, Kd in SHAPES:
        w = (torch.randn(N, Kd, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
        weights[name] = [plugin.pack_weight(w) for _ in range(rot)]
        weights[name + ".bf16"] = w
    xs = {(M, Kd): torch.randn(M, Kd, device=dev, generator=gen).to(torch.bfloat16)
          for M in MS for Kd in {k for _, _, k in SHAPES}}
    log(f"weights: {total_w / 1e6:.0f} MB of digits per copy, {rot} copies")

    ops = [(M, name, N, Kd) for M in MS for name, N, Kd in SHAPES]

    def op_call(M, name, Kd, r):
        return torch.ops.exactmm.linear(xs[(M, Kd)], *weights[name][r])

    # ---------------------------------------------------------------- the step graph
    def step_calls(r):
        # each op uses copy (r + op index) % rot, so consecutive uses of a shape's weights differ
        for i, (M, name, N, Kd) in enumerate(ops):
            op_call(M, name, Kd, (r + i) % rot)

    for r in range(rot):
        step_calls(r)
    torch.cuda.synchronize()
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_calls(0)
    torch.cuda.current_stream().wait_stream(side)
    for r in range(rot):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step_calls(r)
        graphs.append(g)
    for i in range(args.warmup):
        graphs[i % rot].replay()
    torch.cuda.synchronize()
    st, en = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0 = time.perf_counter()
    st.record()
    for i in range(args.steps):
        graphs[i % rot].replay()
    en.record()
    torch.cuda.synchronize()
    wall = time.perf_counter() - t0
    step_ms = st.elapsed_time(en) / args.steps
    step_bytes = sum(gemm_bytes(M, N, Kd) for M, _, N, Kd in ops)
    step_ops = sum(gemm_ops(M, N, Kd) for M, _, N, Kd in ops)
    value = step_bytes / (step_ms * 1e-3) / 1e9
    log(f"step {step_ms:.3f} ms (wall {wall * 1e3 / args.steps:.3f} ms), {value:.1f} GB/s")
    del graphs

    # ---------------------------------------------------------------- per-op detail
    # Each shape is timed on enough weight copies that one rotation streams >= 768 MB, past
    # the 256 MB MALL (three copies of a small shape would stay in it).
    sys.path.insert(0, str(ROOT / "oracle"))
    import oracle  # CPU oracle: checks the outputs, never computes them

    per_op = {}
    for name, N, Kd in SHAPES:
        wd = oracle.digitize_c(weights[name + ".bf16"].float().cpu().numpy(), F)
        nrot = max(rot, rotations_for(2 * N * Kd))
        wc = weights[name] + [tuple(t.clone() for t in weights[name][0]) for _ in range(nrot - rot)]
        wbs = [weights[name + ".bf16"].clone() for _ in range(rotations_for(2 * N * Kd))]
        # the vendor int8 GEMM (torch._int_mm, one int8 dot, int32 out) on the same shape, for
        # scale: the exact path runs three such dots
        b8 = [torch.randint(-128, 128, (N, Kd), dtype=torch.int8, device=dev, generator=gen)
              for _ in range(rotations_for(N * Kd))]
        for M in MS:
            cfg = plugin._cfg(M, N, Kd)
            x = xs[(M, Kd)]
            t_op, t_gemm, one_launch = time_op_and_gemm(torch, K, plugin, x, wc, N, Kd, F, TRUNC, cfg)
            t_bf16 = time_graph(lambda r: torch.matmul(x, wbs[r].T), len(wbs))
            t_i8 = None
            if M > 16:
                a8 = torch.randint(-128, 128, (M, Kd), dtype=torch.int8, device=dev, generator=gen)
                try:
                    t_i8 = round(time_graph(lambda r: torch._int_mm(a8, b8[r].T), len(b8)), 2)
                except RuntimeError:
                    t_i8 = None
            rec = dict(M=M, op=name, N=N, K=Kd, cfg=list(cfg), op_us=round(t_op, 2), gemm_us=round(t_gemm, 2),
                       bf16_hipblaslt_us=round(t_bf16, 2), int8_1dot_vendor_us=t_i8,
                       **roof_fields(M, N, Kd, t_gemm, NDOTS),
                       vs_bf16=round(t_op / t_bf16, 2), weight_copies=nrot, one_launch=one_launch,
                       bit_exact=sampled_rows_exact(torch, np, oracle, x, wd, op_call(M, name, Kd, 0), F, TRUNC))
            per_op[(M, name)] = rec
            log(json.dumps(rec))
        del wc, wbs, b8
        torch.cuda.empty_cache()
    per_op = [per_op[(M, name)] for M, name, _, _ in ops]
    # measured HBM traffic per launch, where the counter record matches these sources and cfg
    op_traffic, op_traffic_note = read_op_traffic()
    for r in per_op:
        t = op_traffic.get((r["M"], r["op"]))
        if t is not None and t[1] == r["cfg"]:
            r["traffic_bytes"] = t[0]
            r["traffic_over_algorithmic"] = round(t[0] / gemm_bytes(r["M"], r["N"], r["K"]), 3)
        else:
            r["traffic_bytes"] = None

    # dominant kernel: the GEMM with the largest share of the step, timed alone on its stream
    dom = max(per_op, key=lambda r: r["gemm_us"])
    M, N, Kd, name = dom["M"], dom["N"], dom["K"], dom["op"]
    cfg = tuple(dom["cfg"])
    xd = K.digitize_packed(xs[(M, Kd)], F)
    nrot = max(rot, rotations_for(2 * N * Kd))
    wc = weights[name] + [tuple(t.clone() for t in weights[name][0]) for _ in range(nrot - rot)]
    out = torch.empty(M, N, device=dev, dtype=torch.bfloat16)  # the op's output dtype
    kstream = torch.cuda.Stream()
    with torch.cuda.stream(kstream):
        # an untimed pass of the same graph first (warm-up, as for the step), then the timing
        for replays in (15, 30):
            t_kernel = time_graph(lambda r: K.exact_linear_packed(xd, (wc[r][0], wc[r][2], wc[r][3]), Kd, F, TRUNC,
                                                                  out=out, cfg=cfg), nrot, calls_per_replay=20,
                                  replays=replays)
    del wc
    b, o = gemm_bytes(M, N, Kd), gemm_ops(M, N, Kd)
    if dom["bound"] == "hbm":
        roof = dict(bound="hbm", achieved=round(b / t_kernel / 1e3, 1), peak=HBM_PEAK_GBS, unit="GB/s",
                    frac=round(b / t_kernel / 1e3 / HBM_PEAK_GBS, 4), traffic=None)
    else:
        roof = dict(bound="mfma", achieved=round(o / t_kernel / 1e6, 1), peak=INT8_PEAK_TOPS, unit="TFLOP/s",
                    frac=round(o / t_kernel / 1e6 / INT8_PEAK_TOPS, 4), traffic=None)
    roof["traffic"], roof["traffic_source"] = (read_traffic(cfg) if (M, name) == (256, "gate_up")
                                               else (None, "no traffic measurement for this kernel"))
    roof.update(kernel=f"exact GEMM M={M} {name} {N}x{Kd} cfg={list(cfg)}", kernel_us=round(t_kernel, 2),
                algorithmic_bytes=b, algorithmic_ops=o)
    log("roofline:", json.dumps(roof))

    # ---------------------------------------------------------------- bit-exactness of the outputs
    # every op of the sweep, on its sampled rows (rows 0..7, M/2 and M-1)
    exact_ok = all(r["bit_exact"] for r in per_op)
    log("bit-exact vs oracle:", exact_ok)

    # ---------------------------------------------------------------- 4 dots: F = 15 sweep, config 1
    per_op_f15, cfg1 = [], None
    if not args.no_f15:
        per_op_f15 = sweep_f15(torch, K, plugin, weights, xs, args.table_f15, args.table, np, oracle)
        cfg1 = config1(torch, K, plugin, oracle, np, dev, gen)

    # ---------------------------------------------------------------- attention
    attn = []
    if not args.no_attention:
        H, KV, D, BS = 32, 8, 128, 16
        P.MAX_LEN = 16384
        for B, L in ATTN_CASES:
            nbp = L // BS
            nblocks = B * nbp
            kv = torch.randn(nblocks, KV, BS, 2 * D, device=dev, generator=gen, dtype=torch.bfloat16)
            bt = torch.randperm(nblocks, device=dev, generator=gen).view(B, nbp).to(torch.int32)
            q = torch.randn(B, H, D, device=dev, generator=gen, dtype=torch.bfloat16)
            sl = torch.full((B,), L, device=dev, dtype=torch.int32)
            kc, vc = kv.transpose(1, 2).split(D, dim=-1)
            out = torch.empty(B, H, D, device=dev, dtype=torch.bfloat16)
            # Three timings of 200 calls each; the last, the steady state, is reported. On some
            # shapes the first 200-400 calls run up to 4 % slower; the first timing is kept as
            # us_first.
            ts = [time_graph(lambda r: P.paged_decode(q, kc, vc, bt, sl, D ** -0.5, out, B, L), 1,
                             calls_per_replay=10, replays=20) for _ in range(3)]
            t = ts[-1]
            kv_bytes = B * L * KV * D * 2 * 2
            rec = dict(B=B, L=L, us=round(t, 2), us_first=round(ts[0], 2), kv_bytes=kv_bytes,
                       TBps=round(kv_bytes / t / 1e6, 3), hbm_frac=round(kv_bytes / t / 1e3 / HBM_PEAK_GBS, 3))
            attn.append(rec)
            log(json.dumps(rec))
            del kv, kc, vc
            torch.cuda.empty_cache()

    # ---------------------------------------------------------------- exact lm_head 4096 -> 151936
    lm_head = []
    if not args.no_lm_head:
        N, Kd = VOCAB, HIDDEN
        w = (torch.randn(N, Kd, device=dev, generator=gen) * 0.02).to(torch.bfloat16)
        lw = [plugin.pack_weight(w) for _ in range(2)]
        for M in (16, 256):
            # activations N(0,1) scaled per row by 10^U(-2,2): mixed magnitudes through the epilogue
            scale = 10.0 ** (torch.rand(M, 1, device=dev, generator=gen) * 4 - 2)
            x = (torch.randn(M, Kd, device=dev, generator=gen) * scale).to(torch.bfloat16)
            t = time_graph(lambda r: torch.ops.exactmm.linear(x, *lw[r]), 2, calls_per_replay=4, replays=10)
            b, o = gemm_bytes(M, N, Kd), gemm_ops(M, N, Kd)
            y = torch.ops.exactmm.linear(x, *lw[0])
            # bit-exactness on sampled rows and the first 4096 vocabulary rows
            rows = np.array([0, M // 2, M - 1])
            wd = oracle.digitize_c(w[:4096].float().cpu().numpy(), F)
            xdn = oracle.digitize_c(x.float().cpu().numpy()[rows], F)
            want = oracle.bf16_rne_c(oracle.exact_linear_c(xdn, wd, F, TRUNC)).reshape(len(rows), 4096)
            got = y[rows.tolist(), :4096].cpu().view(torch.int16).numpy().view(np.uint16)
            rec = dict(M=M, N=N, K=Kd, op_us=round(t, 2), GBps=round(b / t / 1e3, 1), hbm_frac=round(b / t / 1e3 / HBM_PEAK_GBS, 3),
                       TOPS=round(o / t / 1e6, 1), mfma_frac=round(o / t / 1e6 / INT8_PEAK_TOPS, 3),
                       cfg=list(plugin._cfg(M, N, Kd)), bit_exact=bool(np.array_equal(got, want)))
            lm_head.append(rec)
            log(json.dumps(rec))
        del w, lw
        torch.cuda.empty_cache()

    # ---------------------------------------------------------------- decode-step emulation
    decode = []
    if not args.no_decode_step:
        P.MAX_LEN = 16384
        model = DecodeStep(torch, plugin, P, dev, gen)
        log(f"decode-step model: {model.digit_bytes / 1e9:.2f} GB of weight digits")
        for B, L in DECODE_CASES:
            caches, bt, sl = model.kv(B, L, gen)
            h0 = torch.randn(B, HIDDEN, device=dev, generator=gen).to(torch.bfloat16)
            rec = dict(B=B, L=L)
            out = {}

            def whole(exact):
                out["logits"] = model.step(h0, caches, bt, sl, exact)

            parts = model.parts(B, caches, bt, sl, gen)
            for exact in (True, False):
                leg = "exact" if exact else "bf16_hipblaslt"
                rec[leg + "_ms"] = round(graph_ms(torch, lambda: whole(exact)), 3)
                if exact:
                    full = out["logits"].clone()
                out.clear()
                # each part of the step timed on its own (graph replay); the remainder is what
                # the parts do not account for when run back to back in one graph
                br = {name: round(graph_ms(torch, lambda: fn(exact)), 3) for name, fn in parts.items()}
                br["sum_of_parts"] = round(sum(br.values()), 3)
                br["whole_minus_parts"] = round(rec[leg + "_ms"] - br["sum_of_parts"], 3)
                rec[leg + "_breakdown_ms"] = br
            del parts
            # bitwise batch invariance of the exact logits: first and last request alone, and
            # the two of them as a batch in reversed order
            ok = True
            for i in (0, B - 1):
                ok &= torch.equal(model.step(h0[i:i + 1], caches, bt[i:i + 1], sl[i:i + 1]), full[i:i + 1])
            sel = torch.tensor([B - 1, 0], device=dev)
            ok &= torch.equal(model.step(h0[sel], caches, bt[sel].contiguous(), sl[sel].contiguous()), full[sel])
            kv_bytes = len(caches) * B * L * ATT_KV * ATT_D * 2 * 2
            floor_ms = (model.digit_bytes + kv_bytes) / (HBM_PEAK_GBS * 1e9) * 1e3
            rec.update(ratio_exact_vs_bf16=round(rec["exact_ms"] / rec["bf16_hipblaslt_ms"], 3),
                       logits_batch_invariant=bool(ok), hbm_floor_ms=round(floor_ms, 3),
                       exact_hbm_frac=round(floor_ms / rec["exact_ms"], 3))
            decode.append(rec)
            log(json.dumps(rec))
            del caches, bt, sl, full
            torch.cuda.empty_cache()
        del model
        torch.cuda.empty_cache()

    # ---------------------------------------------------------------- CPU baseline (reference CPU path, sampled)
    cpu = None
    if not args.no_cpu:
        del weights
        torch.cuda.empty_cache()
        cpu, cpu_op_s = cpu_baseline_leg(torch, K, np, oracle, step_bytes, ops, args.cpu_seconds)
        if decode:
            # decode step on the CPU, extrapolated: the sampled per-op torch times at M = B,
            # lm_head scaled from QKV by N, attention from a timed fp64 oracle sample
            rng = np.random.default_rng(1)
            Ls = 1024
            qs = rng.standard_normal((1, ATT_H, ATT_D)).astype(np.float32)
            cache = rng.standard_normal((Ls // ATT_BS, ATT_BS, ATT_KV, ATT_D)).astype(np.float32)
            to_bits = lambda a: (a.view(np.uint32) >> 16).astype(np.uint16)
            bt_s = np.arange(Ls // ATT_BS, dtype=np.int32).reshape(1, -1)
            sl_s = np.array([Ls], np.int32)
            t0 = time.perf_counter()
            oracle.paged_decode_c(to_bits(qs), to_bits(cache), to_bits(cache), bt_s, sl_s, ATT_D ** -0.5, 1)
            att_key_s = (time.perf_counter() - t0) / Ls
            for rec in decode:
                B = rec["B"]
                lin_s = LAYERS * sum(cpu_op_s[(B, name)] for name, _, _ in SHAPES)
                lm_s = cpu_op_s[(B, "qkv")] * VOCAB / 6144
                att_s = (LAYERS // ATTN_EVERY) * B * rec["L"] * att_key_s
                rec["cpu_ms_extrapolated"] = round((lin_s + lm_s + att_s) * 1e3, 1)
            log("decode step cpu:", json.dumps([(r["B"], r["L"], r["cpu_ms_extrapolated"]) for r in decode]))

    result = {
        "metric": METRIC,
        "value": round(value, 1),
        "unit": "GB/s",
        "n_gpus": 1,
        "steps": args.steps,
        "warmup": args.warmup,
        "ms_per_step": round(step_ms, 4),
        "higher_is_better": True,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "int8",
        "data": "synthetic",
        "config": {"workload": "decode-shaped exact linear sweep: QKV 4096->6144, O 4096->4096, gate_up "
                               "4096->24576, down 12288->4096 at M in {1,16,64,256}; bf16 in/out, F=14 truncated "
                               "(3 INT8 dots), full exactmm::linear op (digitize + GEMM), weights rotated past MALL",
                   "F": F, "trunc": TRUNC, "step_algorithmic_bytes": step_bytes, "step_int8_ops": step_ops,
                   "step_TOPS": round(step_ops / (step_ms * 1e-3) / 1e12, 2)},
        "roofline": roof,
        "cpu_baseline": cpu,
        "bit_exact": exact_ok and all(r["bit_exact"] for r in per_op_f15 + lm_head)
        and (cfg1 is None or cfg1["bit_exact_fp32_bf16"]),
        "bit_exact_scope": "sampled output rows (0..7, M/2, M-1) of every per_op and per_op_f15 op, rows 0, "
                           "M/2, M-1 of lm_head (first 4096 columns), all of config1 (fp32 and bf16), against the "
                           "CPU oracle",
        "per_op": per_op,
        "per_op_traffic_source": op_traffic_note,
        "per_op_f15": per_op_f15,
        "config1": cfg1,
        "attention": attn,
        "lm_head": lm_head,
        "decode_step": decode,
    }
    print(json.dumps(result), flush=True)


if __name__ == "__main__":
    main()
