"""Measured cases of the serving operators: RMS norm with residual and 8-bit
output, rotary positions, and the matrix-vector product with 4-bit weights.

`listed()` and `draw()` describe cases, `prepare()` makes one case's inputs on
the GPU, `run()` makes one pass: in elementary torch operations, or, with
`own` set, through the library's C entry points (include/tessera_b200_ops.h).
"""
import math
import os
import sys

import torch

own = False

BF16, F16, F32, I8, E4M3, I32, I64 = range(7)  # the library's type codes
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
CODES = {"bf16": BF16, "f16": F16, "f32": F32, "i8": I8, "e4m3": E4M3, "i32": I32, "i64": I64}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "i8": 1, "e4m3": 1}
TOP = {"i8": 127.0, "e4m3": 448.0}
EPS = 1e-6


def listed():
    return [
        # The norm of one new token: nothing but latency.
        {"name": "rms_token", "op": "rms", "M": 1, "D": 640, "pad": 0, "type": "bf16", "res": True, "out": "bf16",
         "group": 0},
        # The head's 2560 columns for a full chunk of pixels, in e4m3 with one scale per pixel.
        {"name": "rms_head", "op": "rms", "M": 32768, "D": 2560, "pad": 0, "type": "bf16", "res": False,
         "out": "e4m3", "group": 0},
        # A full chunk of tokens between two layers: residual stream updated, e4m3 for the next product.
        {"name": "rms_chunk", "op": "rms", "M": 524288, "D": 640, "pad": 0, "type": "bf16", "res": True,
         "out": "e4m3", "group": 128},
        # A width and pitch that no vector load fits, as int8 codes with one scale per row.
        {"name": "rms_odd", "op": "rms", "M": 10007, "D": 1337, "pad": 4, "type": "f16", "res": True, "out": "i8",
         "group": 0},
        # q and k of one pixel's 40-step series, positions = day of year inside the S2 records.
        {"name": "rope_series", "op": "rope", "M": 40, "heads": 8, "hd": 160, "rot": 160, "rest": 640,
         "type": "bf16", "inter": False, "pos": "f32", "stride": 11, "span": 366, "factor": 1.0, "inverse": False},
        # q and k of a full chunk of S1 tokens.
        {"name": "rope_chunk", "op": "rope", "M": 524288, "heads": 8, "hd": 160, "rot": 160, "rest": 640,
         "type": "bf16", "inter": False, "pos": "f32", "stride": 3, "span": 366, "factor": 1.0, "inverse": False},
        # Far positions with frequencies stretched for them, part of each head, grouped k heads, interleaved.
        {"name": "rope_long", "op": "rope", "M": 131071, "heads": 10, "hd": 128, "rot": 64, "rest": 256,
         "type": "bf16", "inter": True, "pos": "i64", "stride": 1, "span": 1000000, "factor": 32.0,
         "inverse": False},
        # Odd head sizes in 32 bits, turned back.
        {"name": "rope_odd", "op": "rope", "M": 5003, "heads": 5, "hd": 51, "rot": 26, "rest": 7, "type": "f32",
         "inter": False, "pos": "i32", "stride": 1, "span": 4096, "factor": 1.0, "inverse": True},
        # The head's first layer for one pixel.
        {"name": "w4_head", "op": "w4", "M": 1, "N": 2560, "K": 1280, "group": 128, "type": "bf16", "xgroup": 0,
         "relu": True, "res": False, "out": "bf16"},
        # QKV of one pixel's series from the norm's 8-bit output.
        {"name": "w4_series", "op": "w4", "M": 40, "N": 1920, "K": 640, "group": 32, "type": "e4m3", "xgroup": 128,
         "relu": False, "res": False, "out": "bf16"},
        # One token against a large matrix.
        {"name": "w4_large", "op": "w4", "M": 1, "N": 16384, "K": 8192, "group": 128, "type": "bf16", "xgroup": 0,
         "relu": False, "res": False, "out": "bf16"},
        # A batch of tokens, ragged in every size, with a residual.
        {"name": "w4_batch", "op": "w4", "M": 17, "N": 8191, "K": 10001, "group": 64, "type": "f16", "xgroup": 0,
         "relu": False, "res": True, "out": "f16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms", "rope", "w4"])
    if op == "rms":
        D = _log(rng, 1, 16384)
        if rng.random() < 0.5:
            D = min(16384, -(-D // 64) * 64)
        out = rng.choice(["same", "i8", "e4m3"])
        t = rng.choice(["bf16", "f16", "f32"])
        M = _log(rng, 1, max(1, min(524288, 524288 * 640 // (2 * D))))
        return {"op": op, "M": M, "D": D, "pad": rng.choice([0, 0, 8, 5]), "type": t, "res": rng.random() < 0.6,
                "out": t if out == "same" else out, "group": 0 if out == "same" else rng.choice([0, 32, 64, 128])}
    if op == "rope":
        heads, hd = rng.randint(1, 48), rng.choice([rng.randint(2, 256), 8 * rng.randint(1, 32)])
        rot = hd // 2 * 2 if rng.random() < 0.5 else 2 * rng.randint(1, hd // 2)
        pos = rng.choice(["f32", "i32", "i64"])
        M = _log(rng, 1, max(1, min(524288, 524288 * 640 // (heads * hd))))
        return {"op": op, "M": M, "heads": heads, "hd": hd, "rot": rot, "rest": rng.choice([0, 0, hd, 3]),
                "type": rng.choice(["bf16", "f16", "f32"]), "inter": rng.random() < 0.5, "pos": pos,
                "stride": rng.choice([1, 3, 11]) if pos == "f32" else 1, "span": _log(rng, 16, 4000000),
                "factor": rng.choice([1.0, 4.0, 32.0]), "inverse": rng.random() < 0.3}
    K = _log(rng, 1, 16384)
    if rng.random() < 0.6:
        K = -(-K // 128) * 128
    t = rng.choice(["bf16", "f16", "i8", "e4m3"])
    return {"op": op, "M": _log(rng, 1, 64), "N": _log(rng, 1, min(16384, 16384 * 8192 // K)), "K": K,
            "group": rng.choice([32, 64, 128]), "type": t,
            "xgroup": rng.choice([0, 32, 64, 128]) if t in TOP else 0, "relu": rng.random() < 0.3,
            "res": rng.random() < 0.3, "out": rng.choice(["bf16", "f16", "f32"])}


def _frequencies(rot, factor):
    """theta_i = 10000^(-2i / rot). Stretched by `factor` over an original span of 8192 positions: frequencies that turn
    less than once over it are divided by the factor, those that turn over 32 times stay, a linear ramp between."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if factor == 1.0:
        return f, 1.0
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*n):
        return torch.randn(*n, device="cuda", generator=g)

    def randint(lo, hi, n, dtype=torch.int64):
        return torch.randint(lo, hi, n, device="cuda", generator=g, dtype=dtype)

    c, s, M = case, {"case": case}, case["M"]
    if c["op"] == "rms":
        D, ld, t = c["D"], c["D"] + c["pad"], TYPES[c["type"]]
        # a residual stream: rows of different size, a few channels that stand out, rows of a padded batch that are zero
        x = randn(M, ld) * torch.exp(0.5 * randn(M, 1))
        x *= 1 + 8 * (torch.rand(ld, device="cuda", generator=g) < 0.01)
        if M >= 64:
            x[M - M // 64:] = 0
        s["x"] = x.to(t)
        if c["res"]:
            r = randn(M, ld)
            if M >= 64:
                r[M - M // 64:] = 0
            s["res"], s["sum"] = r.to(t), torch.zeros(M, ld, device="cuda", dtype=t)
        s["g"] = 1 + 0.1 * randn(D)
        s["y"] = torch.zeros(M, ld, device="cuda", dtype=TYPES[c["out"]])
        if c["out"] in TOP:
            s["scales"] = torch.zeros(M, -(-D // c["group"]) if c["group"] else 1, device="cuda")
            s["values"] = torch.zeros(M, D, device="cuda", dtype=torch.bfloat16) if c["out"] == "i8" else None
    elif c["op"] == "rope":
        width, t = c["heads"] * c["hd"], TYPES[c["type"]]
        s["x"] = randn(M, width + c["rest"]).to(t)  # q and k heads, then what the call leaves alone
        pos = randint(0, c["span"], (M, c["stride"])).sort(0).values
        s["pos"] = pos.to({"f32": torch.float32, "i32": torch.int32, "i64": torch.int64}[c["pos"]])
        f, s["mscale"] = _frequencies(c["rot"], c["factor"])
        s["freq"] = f.cuda()
        s["y"] = torch.zeros(M, width, device="cuda", dtype=t)
    else:
        N, K, G, t = c["N"], c["K"], c["group"], c["type"]
        ng = -(-K // G)
        s["codes"] = randint(-8, 8, (N, K), torch.int8)
        s["wscales"] = ((0.5 + torch.rand(N, ng, device="cuda", generator=g)) / (4.6 * K ** 0.5)).to(torch.bfloat16)
        s["w"] = _packed(s["codes"], s["wscales"], G)
        if t in TOP:
            s["x"] = (randn(M, K) * TOP[t] / 4).clamp(-TOP[t], TOP[t]).to(TYPES[t])
            xg = -(-K // c["xgroup"]) if c["xgroup"] else 1
            s["xscales"] = (0.5 + torch.rand(M, xg, device="cuda", generator=g)) * 4 / TOP[t]
        else:
            s["x"] = randn(M, K).to(TYPES[t])
        s["bias"] = 0.1 * randn(N)
        if c["res"]:
            s["res"] = randn(M, N).to(TYPES[c["out"]])
        s["y"] = torch.zeros(M, N, device="cuda", dtype=TYPES[c["out"]])
    return s


def _packed(codes, scales, G):
    """The library's layout of 4-bit weights: records of 16 rows x 128 columns in the order of its matrix instruction.

    A record holds, for the row halves 0-7 and 8-15, 32 lanes x 16 bytes (lane = 4 row + t; word i of a lane holds columns
    32 i + 8 t .. + 7, the even ones in its low half), then the 128 / G group scales of its 16 rows."""
    N, K = codes.shape
    rt, kb = -(-N // 16), -(-K // 128)
    u = torch.full((rt * 16, kb * 128), 8, dtype=torch.uint8, device=codes.device)
    u[:N, :K] = (codes + 8).view(torch.uint8)
    # rows: tile, half, row; columns: block, word, t, pair, odd
    u = u.view(rt, 2, 8, kb, 4, 4, 2, 2, 2).permute(0, 3, 1, 2, 5, 4, 8, 6, 7)
    # tile, block, half, row, t, word, odd, pair of the half, low / high nibble of its byte
    b = u[..., 0] | u[..., 1] << 4
    b = b.reshape(rt, kb, 1024)
    sc = torch.zeros(rt * 16, kb * (128 // G), dtype=torch.bfloat16, device=codes.device)
    sc[:N, :scales.shape[1]] = scales
    sc = sc.view(rt, 16, kb, 128 // G).permute(0, 2, 3, 1).reshape(rt, kb, -1).contiguous().view(torch.uint8)
    return torch.cat([b, sc], 2).contiguous()


def run(s):
    c = s["case"]
    return {"rms": _rms, "rope": _rope, "w4": _w4}[c["op"]](s, c)


def _library():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tessera-inference_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import tessera_b200
    return tessera_b200.load_library()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _done(rc):
    if rc != 0:
        raise RuntimeError("the call failed")


def _rms(s, c):
    D, ld, y, sc = c["D"], c["D"] + c["pad"], s["y"], s.get("scales")
    if own:
        _done(_library().tcb_op_rmsnorm(
            s["x"].data_ptr(), ld, _ptr(s.get("res")), ld, _ptr(s.get("sum")), ld, s["g"].data_ptr(), EPS,
            CODES[c["type"]], y.data_ptr(), ld, CODES[c["out"]], _ptr(sc), c["group"], c["M"], D,
            torch.cuda.current_stream().cuda_stream))
        y, h = y[:, :D], s["sum"][:, :D] if c["res"] else None
    else:
        h = s["x"][:, :D]
        if c["res"]:
            h = (h.float() + s["res"][:, :D].float()).to(s["x"].dtype)
        v = h.float()
        v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["g"]
        y, sc = _quantised(v, c["out"], c["group"]) if c["out"] in TOP else (v.to(y.dtype), None)
    r = {"y": y}
    if c["res"]:
        r["sum"] = h
    if c["out"] in TOP:
        r["scales"] = sc
        if c["out"] == "i8":  # the values that the codes stand for
            G = c["group"]
            each = sc if not G or sc.shape[1] == 1 else sc.repeat_interleave(G, 1)[:, :D]
            r["y"] = torch.mul(y, each, out=s["values"])
    return r


def _quantised(v, kind, G):
    M, D = v.shape
    G = G or D
    n = -(-D // G)
    p = torch.nn.functional.pad(v, (0, n * G - D)).view(M, n, G)
    sc = p.abs().amax(2).clamp_min(1e-12) / TOP[kind]
    q = (p / sc[:, :, None]).view(M, n * G)[:, :D]
    q = q.round().clamp(-127, 127) if kind == "i8" else q.clamp(-448, 448)
    return q.to(TYPES[kind]), sc


def _rope(s, c):
    M, H, hd, rot = c["M"], c["heads"], c["hd"], c["rot"]
    if own:
        _done(_library().tcb_op_rope(
            s["x"].data_ptr(), s["x"].shape[1], hd, CODES[c["type"]], s["pos"].data_ptr(), c["stride"], CODES[c["pos"]],
            s["freq"].data_ptr(), s["mscale"], rot, int(c["inter"]), int(c["inverse"]), s["y"].data_ptr(), H * hd, hd,
            M, H, hd, torch.cuda.current_stream().cuda_stream))
        return s["y"]
    x = s["x"][:, :H * hd].view(M, H, hd)
    a = s["pos"][:, 0].double()[:, None] * s["freq"]  # far angles need 64 bits
    co, si = (torch.cos(a) * s["mscale"]).float()[:, None], (torch.sin(a) * s["mscale"]).float()[:, None]
    if c["inverse"]:
        si = -si
    p, q = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["inter"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = p.float(), q.float()
    u, v = p * co - q * si, p * si + q * co
    turned = torch.stack((u, v), 3).flatten(2) if c["inter"] else torch.cat((u, v), 2)
    return torch.cat((turned.to(x.dtype), x[..., rot:]), 2).view(M, H * hd)


def _w4(s, c):
    M, N, K, G = c["M"], c["N"], c["K"], c["group"]
    x = s["x"]
    if own:
        _done(_library().tcb_op_gemv_w4(
            x.data_ptr(), K, CODES[c["type"]], _ptr(s.get("xscales")), c["xgroup"], s["w"].data_ptr(), G,
            s["bias"].data_ptr(), int(c["relu"]), _ptr(s.get("res")), N, s["y"].data_ptr(), N, CODES[c["out"]], M, N, K,
            torch.cuda.current_stream().cuda_stream))
        return s["y"]
    w = s["codes"].float() * s["wscales"].float().repeat_interleave(G, 1)[:, :K]
    x = x.float()
    if c["type"] in TOP:
        sc = s["xscales"]
        x = x * (sc.repeat_interleave(c["xgroup"], 1)[:, :K] if c["xgroup"] else sc)
    y = x @ w.t() + s["bias"]
    if c["relu"]:
        y = torch.relu(y)
    if c["res"]:
        y = y + s["res"].float()
    return y.to(s["y"].dtype)


def work(case):
    c, M = case, case["M"]
    if c["op"] == "rms":
        D, t = c["D"], BYTES[c["type"]]
        n = M * D * (t * (3 if c["res"] else 1) + BYTES[c["out"]]) + 4 * D
        if c["out"] in TOP:
            n += 4 * M * (-(-D // c["group"]) if c["group"] else 1)
        return {"bytes": n, "flops": 6 * M * D}
    if c["op"] == "rope":
        n = 2 * M * c["heads"] * c["hd"] * BYTES[c["type"]] + M * (8 if c["pos"] == "i64" else 4) + 4 * c["rot"]
        return {"bytes": n, "flops": 3 * M * c["heads"] * c["rot"]}
    N, K = c["N"], c["K"]
    n = N * K / 2 + 2 * N * -(-K // c["group"]) + M * K * BYTES[c["type"]] + 4 * N
    n += M * N * BYTES[c["out"]] * (2 if c["res"] else 1)
    if c["type"] in TOP:
        n += 4 * M * (-(-K // c["xgroup"]) if c["xgroup"] else 1)
    return {"bytes": n, "flops": 2 * M * N * K}


def exact(case, seed):
    """The definitions in 64 bits. Sums and 8-bit codes are rounded where the definition rounds them."""
    c, s, M = case, prepare(case, seed), case["M"]
    if c["op"] == "rms":
        D = c["D"]
        r, h = {}, s["x"][:, :D].double()
        if c["res"]:
            r["sum"] = (h + s["res"][:, :D].double()).to(s["x"].dtype)
            h = r["sum"].double()
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / D + EPS) * s["g"].double()
        r["y"] = y
        if c["out"] in TOP:
            G = c["group"] or D
            top, sc = TOP[c["out"]], []
            for k in range(0, D, G):
                part = y[:, k:k + G]
                step = part.abs().max(1, keepdim=True).values.clamp(min=1e-12) / top
                sc.append(step)
                part.div_(step)
                if c["out"] == "i8":
                    part.round_().mul_(step)
                else:
                    part.copy_(part.to(torch.float8_e4m3fn))
            r["scales"] = torch.cat(sc, 1)
        return r
    if c["op"] == "rope":
        H, hd, rot = c["heads"], c["hd"], c["rot"]
        y = s["x"][:, :H * hd].double().view(M, H, hd)
        first = torch.arange(0, rot, 2, device="cuda") if c["inter"] else torch.arange(rot // 2, device="cuda")
        second = first + (1 if c["inter"] else rot // 2)
        turn = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device="cuda"),
                           s["pos"][:, 0].double().outer(s["freq"]) * (-1 if c["inverse"] else 1))[:, None]
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y.view(M, H * hd)
    N, K, G = c["N"], c["K"], c["group"]
    y = s["bias"].double().repeat(M, 1)
    x = s["x"].double()
    if c["type"] in TOP:
        at = torch.arange(K, device="cuda") // (c["xgroup"] or K)
        x = x * s["xscales"].double()[:, at]
    for n in range(0, N, 2048):
        w = s["codes"][n:n + 2048].double()
        w *= s["wscales"][n:n + 2048].double()[:, torch.arange(K, device="cuda") // G]
        y[:, n:n + 2048] += x @ w.t()
    if c["relu"]:
        y.clamp_(min=0)
    return y + s["res"].double() if c["res"] else y
