"""Time one back-end kernel alone on a synthetic chunk, through the library's
operator entry points (include/tessera_b200_ops.h), with CUDA events.

  python tessera-inference_b200/op_bench.py attention --T 120        # uniform series of 120 steps
  python tessera-inference_b200/op_bench.py layernorm --M 131072
  python tessera-inference_b200/op_bench.py gemm --M 524288 --N 2560 --K 640 --mode relu --seconds 3 [--torch]
  python tessera-inference_b200/op_bench.py encode --rows 64 --reps 2      # a profiling driver
  python tessera-inference_b200/op_bench.py rmsnorm --M 524288 --D 640 --out e4m3 --group 128
  python tessera-inference_b200/op_bench.py rope --M 524288 --heads 8 --hd 160
  python tessera-inference_b200/op_bench.py gemv --M 1 --N 16384 --K 8192 --group 128

Prints one JSON line: microseconds per launch, the algorithmic bytes of the
launch and the bandwidth they give. Attention bytes per token are the Q, K and
V rows read (3 x 640 bf16) and the output row written (640 bf16): 5,120 B.
LayerNorm bytes per row are 640 bf16 read and written: 2,560 B. Inputs are
seeded random bf16 in device memory, larger than L2 at the default sizes.
`TC_ATTN_TC=2` selects the tcgen05 attention kernel for every series of up
to 128 steps and `TC_ATTN_TC=0` the mma.sync kernel; unset, the library
takes tcgen05 for series longer than 48 steps and up to 128.

The chunk is described by its series length alone (no offsets array), so the
entry point does no host work and the launches run back to back.

`gemm` times the tcgen05 GEMM on one layer shape (mode: bias, relu = bias +
ReLU, res = bias + residual) for about --seconds of back-to-back launches, so
the clock settles under the power cap, and reports TFLOP/s with the median
SM clock sampled by nvidia-smi over the timed loop (and TFLOP/s per GHz).
--torch times torch.matmul (cuBLAS, bf16, no epilogue) on the same shape the
same way, as a comparison point; it is not part of the back end.

`rmsnorm` (bf16 rows with a residual), `rope` (bf16 heads, positions = day of
year) and `gemv` (4-bit weights, bf16 rows) time the token-stream operators. Their
launches go over --sets sets of buffers in turn inside a CUDA graph, so host time
is not in the figure and, with enough sets, nothing is found in L2.

`encode` runs the whole device path (tc_encode_tile_device) --reps times on
a seeded tile of --rows rows with config 1's width, series lengths and value
distributions (synth.make_tile), so every kernel of the path launches at
config-1 chunk sizes; it is the small workload the ncu captures run.
"""
from __future__ import annotations

import argparse
import json
import statistics
import subprocess
import sys
import tempfile
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
import tessera_b200 as tb  # noqa: E402


def time_launches(fn, reps: int) -> float:
    """Microseconds per launch over `reps` launches after three warm-up ones."""
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(reps):
        fn()
    e1.record()
    torch.cuda.synchronize()
    return e0.elapsed_time(e1) * 1e3 / reps


class SmClocks:
    """Median SM clock (MHz) of the current GPU while the block runs (nvidia-smi, 100 ms samples)."""

    def __enter__(self):
        self.f = tempfile.TemporaryFile(mode="w+")
        uuid = str(torch.cuda.get_device_properties(torch.cuda.current_device()).uuid)
        gpu = uuid if uuid.startswith("GPU-") else f"GPU-{uuid}"
        try:
            self.p = subprocess.Popen(["nvidia-smi", "--query-gpu=clocks.sm,power.draw", "--format=csv,noheader,nounits",
                                       "-lms", "100", "-i", gpu], stdout=self.f, stderr=subprocess.DEVNULL)
        except FileNotFoundError:
            self.p = None
        time.sleep(0.2)
        return self

    def __exit__(self, *exc):
        if self.p is not None:
            self.p.terminate()
            self.p.wait(5)

    def median(self):
        self.f.seek(0)
        v = []
        for line in self.f.read().splitlines():
            try:
                mhz, w = (float(x) for x in line.split(","))
            except ValueError:
                continue
            if w > 300:
                v.append(mhz)
        return statistics.median(v) if v else None


def time_for(fn, seconds: float) -> tuple[float, int, float | None]:
    """(microseconds per launch, launches, median SM MHz) over about `seconds`."""
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    fn()
    torch.cuda.synchronize()
    reps = max(3, int(seconds / max(time.perf_counter() - t0, 1e-6)))
    with SmClocks() as clk:
        us = time_launches(fn, reps)
    return us, reps, clk.median()


def time_graph(fns, reps: int) -> float:
    """Microseconds per launch over `reps` rounds of the launches `fns`, replayed as one CUDA graph."""
    for f in fns:
        f(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in fns:
            f(torch.cuda.current_stream().cuda_stream)
    return time_launches(graph.replay, reps) / len(fns)


def token_op(lib, a, g):
    """(operator, launches, algorithmic bytes of one, sizes) of the token-stream operator that `a` names."""
    def randn(*n):
        return torch.randn(*n, device="cuda", generator=g)

    def ok(rc):
        if rc != 0:
            raise RuntimeError(f"{a.op} failed")

    fns, M, D, N, K = [], a.M, a.D, a.N, a.K
    if a.op == "rmsnorm":
        ytype = {"bf16": tb.BF16, "i8": tb.I8, "e4m3": tb.E4M3}[a.out]
        group = a.group if a.out != "bf16" else 0
        ng = -(-D // group) if group else 1
        gam = 1 + 0.1 * randn(D)
        for _ in range(a.sets):
            x, r = randn(M, D).to(torch.bfloat16), randn(M, D).to(torch.bfloat16)
            h, y = torch.empty_like(x), torch.empty(M, D * (2 if a.out == "bf16" else 1), device="cuda", dtype=torch.uint8)
            sc = torch.empty(M, ng, device="cuda")
            fns.append(lambda st, x=x, r=r, h=h, y=y, sc=sc: ok(lib.tcb_op_rmsnorm(
                x.data_ptr(), D, r.data_ptr(), D, h.data_ptr(), D, gam.data_ptr(), 1e-6, tb.BF16, y.data_ptr(), D, ytype,
                sc.data_ptr() if a.out != "bf16" else None, group, M, D, st)))
        nbytes = M * D * (8 if a.out == "bf16" else 7) + (4 * M * ng if a.out != "bf16" else 0)
        return fns, nbytes, {"M": M, "D": D, "out": a.out, "group": group}
    if a.op == "rope":
        width = a.heads * a.hd
        freq = torch.from_numpy(tb.rope_freqs(a.rot or a.hd)[0]).cuda()
        for _ in range(a.sets):
            x = randn(M, width).to(torch.bfloat16)
            y, pos = torch.empty_like(x), torch.randint(1, 367, (M,), device="cuda", generator=g).float()
            fns.append(lambda st, x=x, y=y, pos=pos: ok(lib.tcb_op_rope(
                x.data_ptr(), width, a.hd, tb.BF16, pos.data_ptr(), 1, tb.F32, freq.data_ptr(), 1.0, a.rot or a.hd,
                int(a.interleaved), 0, y.data_ptr(), width, a.hd, M, a.heads, a.hd, st)))
        return fns, 4 * M * width, {"M": M, "heads": a.heads, "hd": a.hd, "rot": a.rot or a.hd, "interleaved": a.interleaved}
    group = a.group or 128
    nb = lib.tcb_w4_bytes(N, K, group)
    if nb < 0:
        raise RuntimeError("bad sizes")
    for _ in range(a.sets):
        # any bytes are codes; scales of 2^-8 (bf16 0x3b80) behind each record's 1,024 bytes
        w = torch.randint(0, 256, (nb,), device="cuda", generator=g, dtype=torch.uint8)
        w.view(-1, 1024 + 4096 // group)[:, 1024:].view(torch.int16).fill_(0x3b80)
        x, y = randn(M, K).to(torch.bfloat16), torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        fns.append(lambda st, w=w, x=x, y=y: ok(lib.tcb_op_gemv_w4(
            x.data_ptr(), K, tb.BF16, None, 0, w.data_ptr(), group, None, 0, None, 0, y.data_ptr(), N, tb.BF16, M, N, K, st)))
    return fns, N * K // 2 + 2 * N * -(-K // group) + 2 * M * (N + K), {"M": M, "N": N, "K": K, "group": group}


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("op", choices=["attention", "layernorm", "gemm", "encode", "rmsnorm", "rope", "gemv"])
    ap.add_argument("--rows", type=int, default=64, help="tile rows (encode)")
    ap.add_argument("--N", type=int, default=2560)
    ap.add_argument("--K", type=int, default=640)
    ap.add_argument("--mode", choices=["bias", "relu", "res"], default="relu")
    ap.add_argument("--variant", type=int, default=0, help="0 per-layer choice, 1 single CTA, 2 CTA pair, 3 operand-swapped")
    ap.add_argument("--seconds", type=float, default=3.0)
    ap.add_argument("--torch", action="store_true", help="also time torch.matmul (cuBLAS) on the same shape")
    ap.add_argument("--T", type=int, default=120, help="uniform series length (attention)")
    ap.add_argument("--tokens", type=int, default=131072, help="tokens per attention chunk")
    ap.add_argument("--M", type=int, default=131072, help="rows (layernorm, rmsnorm, rope, gemv)")
    ap.add_argument("--D", type=int, default=640, help="columns (rmsnorm)")
    ap.add_argument("--out", choices=["bf16", "i8", "e4m3"], default="e4m3", help="output (rmsnorm)")
    ap.add_argument("--group", type=int, default=0, help="columns per scale (rmsnorm: 0 = the row; gemv: 0 = 128)")
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--hd", type=int, default=160)
    ap.add_argument("--rot", type=int, default=0, help="turned columns of a head (rope: 0 = all)")
    ap.add_argument("--interleaved", action="store_true", help="pairs (2i, 2i + 1) (rope)")
    ap.add_argument("--sets", type=int, default=3, help="sets of buffers (rmsnorm, rope, gemv)")
    ap.add_argument("--reps", type=int, default=10)
    a = ap.parse_args(argv)
    lib = tb.load_library()
    st = torch.cuda.current_stream().cuda_stream
    g = torch.Generator(device="cuda").manual_seed(0)
    if a.op == "attention":
        npix = a.tokens // a.T
        M = npix * a.T
        qkv = torch.randn(M, 1920, device="cuda", generator=g).to(torch.bfloat16)
        att = torch.empty(M, 640, device="cuda", dtype=torch.bfloat16)

        def run():
            if lib.tcb_op_attention(qkv.data_ptr(), None, a.T, npix, a.T, att.data_ptr(), st):
                raise RuntimeError("tcb_op_attention failed")

        us = time_launches(run, a.reps)
        nbytes = M * 5120
        rec = {"op": "attention", "tokens": M, "pixels": npix, "T": a.T}
    elif a.op in ("rmsnorm", "rope", "gemv"):
        fns, nbytes, rec = token_op(lib, a, g)
        us = time_graph(fns, a.reps)
        rec = {"op": a.op, **rec}
    elif a.op == "encode":
        import tempfile as tf
        import synth
        tile = synth.make_tile(H=a.rows, W=695, T2=120, Ta=60, Td=60, p=0.6, seed=2)
        T2, H, W = tile["masks"].shape
        with tf.TemporaryDirectory() as td:
            enc = tb.Encoder(synth.make_weights(Path(td) / "w.tcw", seed=0))
        dev = {k: torch.from_numpy(v).cuda() for k, v in tile.items()}
        codes = torch.empty((H, W, 128), dtype=torch.int8, device="cuda")
        scales = torch.empty((H, W), dtype=torch.float32, device="cuda")
        enc.set_stream(st)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for i in range(a.reps):
            if i == a.reps - 1:
                e0.record()
            enc.encode_tile_device(dev, T2, 60, 60, H, W, 0, H, codes, scales)
        e1.record()
        torch.cuda.synchronize()
        ms = e0.elapsed_time(e1)
        enc.close()
        print(json.dumps({"op": "encode", "pixels": H * W, "ms_last": round(ms, 2), "px_s": round(H * W / ms * 1e3)}))
        return 0
    elif a.op == "gemm":
        M, N, K = a.M, a.N, a.K
        A = torch.randn(M, K, device="cuda", generator=g).to(torch.bfloat16)
        W = (torch.randn(N, K, device="cuda", generator=g) / K ** 0.5).to(torch.bfloat16)
        bias = torch.randn(N, device="cuda", generator=g) * 0.1
        res = torch.randn(M, N, device="cuda", generator=g).to(torch.bfloat16) if a.mode == "res" else None
        out = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")

        def run():
            if lib.tcb_op_gemm(A.data_ptr(), K, W.data_ptr(), bias.data_ptr(), int(a.mode == "relu"),
                               res.data_ptr() if res is not None else None, N, None, 1, None, None, out.data_ptr(), N,
                               M, N, K, 0, a.variant, status.data_ptr(), st):
                raise RuntimeError("tcb_op_gemm failed")

        us, reps, mhz = time_for(run, a.seconds)
        torch.cuda.synchronize()
        if status.item() != 0:
            raise RuntimeError(f"device status {status.item()}")
        flop = 2.0 * M * N * K
        rec = {"op": "gemm", "M": M, "N": N, "K": K, "mode": a.mode, "variant": a.variant,
               "us_per_launch": round(us, 2), "TFLOP_s": round(flop / us / 1e6, 1), "sm_mhz": mhz,
               "TFLOP_s_per_GHz": round(flop / us / 1e6 / (mhz / 1e3), 1) if mhz else None, "reps": reps}
        if a.torch:
            Wt = W.t()

            def run_t():
                torch.matmul(A, Wt, out=out)

            us_t, reps_t, mhz_t = time_for(run_t, a.seconds)
            rec["cublas"] = {"us_per_launch": round(us_t, 2), "TFLOP_s": round(flop / us_t / 1e6, 1), "sm_mhz": mhz_t,
                             "TFLOP_s_per_GHz": round(flop / us_t / 1e6 / (mhz_t / 1e3), 1) if mhz_t else None,
                             "reps": reps_t, "what": "torch.matmul bf16, no epilogue"}
        print(json.dumps(rec))
        return 0
    else:
        M = a.M
        x = torch.randn(M, 640, device="cuda", generator=g).to(torch.bfloat16)
        y = torch.empty_like(x)
        gam = torch.ones(640, device="cuda")
        bet = torch.zeros(640, device="cuda")

        def run():
            if lib.tcb_op_layernorm640(x.data_ptr(), M, gam.data_ptr(), bet.data_ptr(), y.data_ptr(), st):
                raise RuntimeError("tcb_op_layernorm640 failed")

        us = time_launches(run, a.reps)
        nbytes = M * 2560
        rec = {"op": "layernorm640", "rows": M}
    rec.update({"us_per_launch": round(us, 2), "bytes_per_launch": nbytes, "GB_per_s": round(nbytes / us / 1e3, 1),
                "reps": a.reps})
    print(json.dumps(rec))
    return 0


if __name__ == "__main__":
    sys.exit(main())
