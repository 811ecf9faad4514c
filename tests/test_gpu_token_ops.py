"""The token-stream operators against their definitions in 64 bits.

Tolerances, derived for each output (H = half a step of its type relative to
the value: bf16 2^-8, fp16 2^-11, f32 2^-24, e4m3 2^-4; an expectation that is
rounded too costs a second H; U = 2^-24, one f32 rounding):

* RMS norm. A row's squares are summed by threads of at most 64 terms each and
  a tree of at most 14 levels, all non-negative: (64 + 14 + 1) U. The root
  halves it; the root, two divisions and three products add 6 U: v is within
  46 U, taken as 64 U. Codes: v / s is within 130 U of its value, at most 127
  (448): 0.5 + 127 * 130 U < 0.5 + 1e-3 from the code (e4m3: H of it, or half
  the smallest step, 2^-10, and 130 U of it).
* Rotary positions. The fraction of a turn is held to 2^-26 turns, an angle of
  2 pi 2^-26 < 2 U; sine and cosine are within 4 U; mscale, product and sum add
  3 U: (|a| + |b|) |mscale| 10 U, plus H of the result.
* 4-bit product. Every product of a code, at most 8, and an x of at most 11
  bits is exact in f32. A sum in any order of n = K terms with one extra
  rounding per group and scale is within (K + 2 K / 32 + 16) U of the sum of
  magnitudes in the worst case; the matrix instruction may truncate where it
  adds, which doubles U. The magnitudes are summed in the test.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import tessera_b200 as tb  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPE = {tb.BF16: torch.bfloat16, tb.F16: torch.float16, tb.F32: torch.float32, tb.I8: torch.int8,
        tb.E4M3: torch.float8_e4m3fn, tb.I32: torch.int32, tb.I64: torch.int64}
HALF = {tb.BF16: 2.0 ** -8, tb.F16: 2.0 ** -11, tb.F32: 2.0 ** -24}
TINY = {tb.BF16: 2.0 ** -133, tb.F16: 2.0 ** -24, tb.F32: 2.0 ** -149}  # smallest subnormal
TOP = {tb.I8: 127.0, tb.E4M3: 448.0}


@pytest.fixture(scope="module")
def lib():
    return tb.load_library()


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *n):
    return torch.randn(*n, device="cuda", generator=g)


def within(got, want, tol):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want) & (got != want)  # equal infinities are equal
    err = (got - want).abs()
    bad = fine & ~(err <= tol)
    assert not bad.any(), f"{bad.sum().item()} of {bad.numel()} out of tolerance; worst {(err - tol)[bad].max().item()}"


# ------------------------------------------------------------------ RMS norm
def rms_ref(x, res, g, eps):
    """(h, v) in the definition: h rounded to x's type, v in f64."""
    h = x if res is None else (x.double() + res.double()).to(x.dtype)
    d = h.double()
    v = d / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    return h, v if g is None else v * g.double()


def check_rms(h, v, y, ytype, group, scales):
    M, D = v.shape
    if ytype not in TOP:
        return within(y, v.to(TYPE[ytype]), v.abs() * (HALF[ytype] * 2 + 64 * U) + TINY[ytype])
    G = group or D
    for k, c in enumerate(range(0, D, G)):
        part, code = v[:, c:c + G], y[:, c:c + G].double()
        amax = part.abs().amax(1)
        s = torch.where(torch.isnan(amax), amax, amax.clamp(min=1e-12)) / TOP[ytype]
        within(scales[:, k], s, s * 80 * U)
        q = part / s[:, None]
        if ytype == tb.I8:
            assert not code[torch.isnan(q)].any()
            within(torch.where(torch.isnan(q), q, code), q, 0.5 + 1e-3)
        else:
            within(code, q, q.abs() * (2.0 ** -4 + 130 * U) + 2.0 ** -10)
    assert scales.shape[1] == -(-D // G)


def run_rms(lib, x, res, g, D, dtype, ytype, group, eps=1e-6, pad=0, want_sum=True, ldy=None):
    """One call on rows of pitch D + pad; checks that nothing between the rows or behind them is written."""
    M, ld = x.shape[0], D + pad
    ldy = ldy or ld
    y = torch.full((M + 1, ldy), 77, device="cuda").to(TYPE[ytype])
    sm = torch.full((M + 1, ld), 77, device="cuda").to(TYPE[dtype]) if res is not None and want_sum else None
    ng = -(-D // group) if group else 1
    sc = torch.full((M + 1, ng), 77.0, device="cuda") if ytype in TOP else None
    assert lib.tcb_op_rmsnorm(_p(x), x.stride(0), _p(res), res.stride(0) if res is not None else 0, _p(sm), ld, _p(g), eps,
                              dtype, _p(y), ldy, ytype, _p(sc), group, M, D, _stream()) == 0
    torch.cuda.synchronize()
    mark = torch.tensor([77.0]).to(TYPE[ytype]).float().item()
    assert (y[M].float() == mark).all() and (y[:, D:].float() == mark).all()
    if sm is not None:
        assert (sm[M] == 77).all() and (sm[:, D:] == 77).all()
        sm = sm[:M, :D]
    if sc is not None:
        assert (sc[M] == 77).all()
        sc = sc[:M]
    return y[:M, :D], sm, sc


def rms_case(lib, M, D, pad, dtype, ytype, group, res, gamma=True, seed=0):
    g = _gen(seed + M * 7 + D)
    x = (_randn(g, M, D + pad) * torch.exp(_randn(g, M, 1))).to(TYPE[dtype])
    r = _randn(g, M, D + pad).to(TYPE[dtype]) if res else None
    w = 1 + 0.2 * _randn(g, D) if gamma else None
    if M > 2:
        x[M // 2] = 0
        if res:
            r[M // 2] = 0
    y, sm, sc = run_rms(lib, x, r, w, D, dtype, ytype, group, pad=pad)
    h, v = rms_ref(x[:, :D], None if r is None else r[:, :D], w, 1e-6)
    if res:
        assert torch.equal(sm, h)
    check_rms(h, v, y, ytype, group, sc)
    if M > 2 and ytype in TOP:  # a row of zeros
        assert not y[M // 2].float().any() and (sc[M // 2] == np.float32(1e-12) / np.float32(TOP[ytype])).all()


SIZES = [(1, 1), (3, 2), (5, 7), (4, 31), (4, 32), (7, 33), (9, 96), (3, 127), (33, 128), (5, 200), (130, 640), (7, 641),
         (6, 1000), (5, 1024), (3, 1032), (5, 1337), (4, 2048), (3, 2560), (2, 4096), (2, 4104), (2, 8191), (2, 8192),
         (2, 16383), (1, 16384)]


@pytest.mark.parametrize("M,D", SIZES)
@pytest.mark.parametrize("dtype", [tb.BF16, tb.F16, tb.F32])
def test_rmsnorm_same_type(lib, M, D, dtype):
    rms_case(lib, M, D, 0, dtype, dtype, 0, True)
    rms_case(lib, M, D, 5, dtype, dtype, 0, False, gamma=False)


@pytest.mark.parametrize("M,D", SIZES)
@pytest.mark.parametrize("ytype", [tb.I8, tb.E4M3])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
def test_rmsnorm_codes(lib, M, D, ytype, group):
    rms_case(lib, M, D, 0, tb.BF16, ytype, group, True)
    rms_case(lib, M, D, 3, tb.F16, ytype, group, False)
    rms_case(lib, M, D, 8, tb.F32, ytype, group, True, gamma=False)


@pytest.mark.parametrize("D", [8, 15, 16, 17, 57, 64, 65, 249, 250, 256, 257, 505, 512, 513, 520, 640, 648, 761, 768, 1017, 1018, 1024, 1025, 1530,
                               1536, 1537, 2041, 2048, 2049, 2560, 2561, 2800, 4089, 4097, 8186, 8193, 16377, 16378])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_rmsnorm_team_edges(lib, D, pad):
    """Widths around the ends of every team, in rows that start on and off the boundaries."""
    rms_case(lib, 5, D, pad, tb.BF16, tb.E4M3, 64, True, seed=pad)
    rms_case(lib, 5, D, pad, tb.F32, tb.F32, 0, True, seed=pad)
    rms_case(lib, 5, D, pad, tb.F16, tb.I8, 0, False, seed=pad)


@pytest.mark.parametrize("D,ld", [(640, 640), (1337, 1341), (100, 103), (2560, 2560)])
@pytest.mark.parametrize("shift", [(1, 1, 1, 1), (3, 3, 3, 3), (1, 0, 0, 0), (0, 2, 5, 0), (0, 0, 0, 1)])
@pytest.mark.parametrize("ytype", [tb.BF16, tb.I8])
def test_rmsnorm_shifted_pointers(lib, D, ld, shift, ytype):
    """x, res, sum and y that start any number of elements behind a boundary, alike or not."""
    g, M, n = _gen(11), 21, 21 * ld + 8
    bufs = [_randn(g, n).to(torch.bfloat16) for _ in range(3)] + [torch.zeros(n, device="cuda", dtype=TYPE[ytype])]
    x, r, sm, y = (b[k:k + M * ld].view(M, ld) for b, k in zip(bufs, shift))
    w = 1 + 0.1 * _randn(g, D + 1)[1:]
    group = 32 if ytype == tb.I8 else 0
    sc = torch.zeros(M, -(-D // group), device="cuda") if group else None
    h, v = rms_ref(x[:, :D], r[:, :D], w, 1e-6)
    edges = [b.clone() for b in bufs]
    assert lib.tcb_op_rmsnorm(_p(x), ld, _p(r), ld, _p(sm), ld, _p(w), 1e-6, tb.BF16, _p(y), ld, ytype, _p(sc), group, M, D,
                              _stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(sm[:, :D], h)
    check_rms(h, v, y[:, :D], ytype, group, sc)
    for b, old, k, written in zip(bufs, edges, shift, (0, 0, 1, 1)):
        if written:
            b[k:k + M * ld].view(M, ld)[:, :D] = old[k:k + M * ld].view(M, ld)[:, :D]
        assert torch.equal(b, old)


@pytest.mark.parametrize("D,dtype", [(641, tb.BF16), (99, tb.F32), (3001, tb.F16)])
def test_rmsnorm_in_place_off_boundaries(lib, D, dtype):
    """All in place, on rows next to one another: a row's ends share 16 bytes with its neighbours' rows."""
    g = _gen(12)
    x, r = _randn(g, 300, D).to(TYPE[dtype]), _randn(g, 300, D).to(TYPE[dtype])
    h, v = rms_ref(x, r, None, 1e-6)
    assert lib.tcb_op_rmsnorm(_p(x), D, _p(r), D, _p(r), D, None, 1e-6, dtype, _p(x), D, dtype, None, 0, 300, D, _stream()) == 0
    assert torch.equal(r, h)
    check_rms(h, v, x, dtype, 0, None)


def test_rmsnorm_row_alone(lib):
    """A row's bits are the same alone and in a long stream."""
    g = _gen(20)
    for D, group in ((640, 128), (37, 32), (64, 0), (1337, 0), (2560, 64), (9000, 0)):
        x = _randn(g, 5000, D).to(torch.bfloat16)
        y, _, sc = run_rms(lib, x, None, None, D, tb.BF16, tb.E4M3, group)
        for r in (0, 1, 2499, 4999):
            start = x[r].data_ptr() // 2 % 8  # where the row starts in the stream
            one = torch.zeros(1, D + 16, device="cuda", dtype=torch.bfloat16)
            z = torch.zeros(D + 16, device="cuda", dtype=torch.uint8)
            s = torch.zeros_like(sc[:1])
            at = (start - one.data_ptr() // 2) % 8
            k = (at + one.data_ptr() // 2 - z.data_ptr()) % 8
            one[0, at:at + D] = x[r]
            assert lib.tcb_op_rmsnorm(one[0, at:].data_ptr(), D, None, 0, None, 0, None, 1e-6, tb.BF16, z[k:].data_ptr(), D,
                                      tb.E4M3, _p(s), group, 1, D, _stream()) == 0
            assert torch.equal(z[k:k + D], y[r].view(torch.uint8)) and torch.equal(s[0], sc[r])


def test_rmsnorm_sums_far_apart(lib):
    """The residual's sum is rounded once, subnormals, infinities and sums past the type's end included."""
    for dtype, vals in ((tb.BF16, [1e-40, 3e-39, 1.0, 257.0, 3e38, float("inf"), -0.0, 1e-3]),
                        (tb.F16, [6e-8, 1e-6, 1.0, 2049.0, 65000.0, float("inf"), -0.0, 1e-3]),
                        (tb.F32, [1e-44, 1e-39, 1.0, 16777217.0, 3e38, float("inf"), -0.0, 1e-3])):
        v = torch.tensor(vals, device="cuda").to(TYPE[dtype])
        x = torch.cat([v[:, None].expand(8, 8), v[:, None].expand(8, 8)], 1).contiguous()
        r = torch.cat([v[None].expand(8, 8), -v[None].expand(8, 8)], 1).contiguous()
        _, sm, _ = run_rms(lib, x, r, None, 16, dtype, dtype, 0)
        want = (x.double() + r.double()).to(TYPE[dtype])
        assert torch.equal(torch.isnan(sm), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(sm, 7.0), torch.nan_to_num(want, 7.0))


def test_rmsnorm_without_eps(lib):
    """eps 0: rows far below 1 are normalised all the same; a row of zeros has no norm."""
    g = _gen(13)
    x = _randn(g, 4, 640)
    x[0] *= 1e-30
    x[1] *= 1e-37
    x[2] = 0
    for dtype in (tb.BF16, tb.F32):
        xt = x.to(TYPE[dtype])
        for ytype, group in ((dtype, 0), (tb.I8, 0), (tb.E4M3, 128)):
            y, _, sc = run_rms(lib, xt, None, None, 640, dtype, ytype, group, eps=0.0)
            h, v = rms_ref(xt, None, None, 0.0)
            check_rms(h, v, y, ytype, group, sc)


def test_rmsnorm_long(lib):
    """More rows than any grid holds at once."""
    rms_case(lib, 70001, 640, 0, tb.BF16, tb.E4M3, 128, True)
    rms_case(lib, 40003, 88, 0, tb.F16, tb.I8, 32, True)


@pytest.mark.parametrize("D", [640, 641, 2560, 5001])
@pytest.mark.parametrize("ytype", [tb.BF16, tb.I8, tb.E4M3])
def test_rmsnorm_far_values(lib, D, ytype):
    """Rows whose squares overflow f32, NaN and infinities, and rows that eps alone holds up."""
    g = _gen(3)
    x = _randn(g, 6, D)
    x[0] *= 1e37
    x[1] *= 1e-30
    x[2, D // 2] = float("nan")
    x[3, 1] = float("inf")
    x[4, D - 1] = float("-inf")
    x = x.to(torch.bfloat16)
    group = 0 if ytype == tb.BF16 else 64
    y, _, sc = run_rms(lib, x, None, None, D, tb.BF16, ytype, group)
    d = x.double()
    v = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-6)
    v[1] = d[1] * 1e3  # sqrt(1e-6 + 1e-60) in f32 and f64 alike
    check_rms(None, v, y, ytype, group, sc)


@pytest.mark.parametrize("D,dtype", [(640, tb.BF16), (1337, tb.F16), (2560, tb.F32)])
def test_rmsnorm_in_place(lib, D, dtype):
    """sum may be x or res, y may be x or sum."""
    g = _gen(4)
    x0, r0 = _randn(g, 50, D).to(TYPE[dtype]), _randn(g, 50, D).to(TYPE[dtype])
    h, v = rms_ref(x0, r0, None, 1e-5)
    for which in ("sum=x", "sum=res", "y=x", "y=sum"):
        x, r, s, y = x0.clone(), r0.clone(), torch.empty_like(x0), torch.empty_like(x0)
        s = x if which == "sum=x" else r if which == "sum=res" else s
        y = x if which == "y=x" else s if which == "y=sum" else y
        assert lib.tcb_op_rmsnorm(_p(x), D, _p(r), D, None if which == "y=sum" else _p(s), D, None, 1e-5, dtype, _p(y), D,
                                  dtype, None, 0, 50, D, _stream()) == 0
        check_rms(h, v, y, dtype, 0, None)
        if which != "y=sum":
            assert torch.equal(s, h) or which == "y=x" and torch.equal(s, h)


def test_rmsnorm_far_pitch(lib):
    """Row offsets beyond 2^31 elements."""
    D, ld = 640, 1_300_000_003
    buf = torch.empty(2 * ld + D, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, D), (ld, 1))
    x.copy_(_randn(_gen(5), 3, D))
    y, _, sc = run_rms(lib, x, None, None, D, tb.BF16, tb.E4M3, 0)
    h, v = rms_ref(x, None, None, 1e-6)
    check_rms(h, v, y, tb.E4M3, 0, sc)


@pytest.mark.parametrize("D", [8, 640, 2560, 5001, 16384])
@pytest.mark.parametrize("dtype", [tb.BF16, tb.F32])
def test_rmsnorm_small_values_in_far_rows(lib, D, dtype):
    """Rows whose squares overflow f32 keep every bit of their small values: each output is within the same relative bound."""
    g = _gen(26)
    x = _randn(g, 6, D) * torch.exp2(100 * torch.rand(6, D, device="cuda", generator=g) - 40)
    x[:, 3] = torch.tensor([2.0 ** 70, 2.0 ** 80, 2.0 ** 64, 2.0 ** 100, 1.5 * 2.0 ** 127, 1.0], device="cuda")
    x, w = x.to(TYPE[dtype]), 1 + 0.2 * _randn(g, D)
    y, _, _ = run_rms(lib, x, None, w, D, dtype, dtype, 0)
    _, v = rms_ref(x, None, w, 1e-6)
    check_rms(None, v, y, dtype, 0, None)
    z, _, sc = run_rms(lib, x, None, w, D, dtype, tb.E4M3, 32)
    check_rms(None, v, z, tb.E4M3, 32, sc)


@pytest.mark.parametrize("dtype", [tb.BF16, tb.F32])
def test_rmsnorm_largest_eps(lib, dtype):
    """mean(h^2) + eps past f32's end, each within it."""
    for D, h, eps in ((1, 1.8e19, 3e38), (2, 1.2e19, 3e38), (2, 1.2e19, 3.4e38), (64, 2.2e18, 3.39e38), (64, 1.0, 3.4e38), (1, 1e-20, 3.4e38)):
        x = torch.full((3, D), h, device="cuda").to(TYPE[dtype])
        x[1] *= -1
        y, _, _ = run_rms(lib, x, None, None, D, dtype, dtype, 0, eps=eps)
        _, v = rms_ref(x, None, None, float(np.float32(eps)))
        check_rms(None, v, y, dtype, 0, None)


@pytest.mark.parametrize("D", [640, 641, 2560, 9001])
def test_rmsnorm_all_over_res(lib, D):
    """sum may be res and y may be sum, so y over res: the norm stands where the residual was."""
    g = _gen(27)
    x, r = _randn(g, 50, D).to(torch.bfloat16), _randn(g, 50, D).to(torch.bfloat16)
    _, v = rms_ref(x, r, None, 1e-5)
    assert lib.tcb_op_rmsnorm(_p(x), D, _p(r), D, _p(r), D, None, 1e-5, tb.BF16, _p(r), D, tb.BF16, None, 0, 50, D, _stream()) == 0
    check_rms(None, v, r, tb.BF16, 0, None)


@pytest.mark.parametrize("D,ld,dtype", [(1337, 1341, tb.F16), (641, 641, tb.BF16), (99, 101, tb.F32)])
def test_rmsnorm_same_row_elsewhere(lib, D, ld, dtype):
    """Rows that are alike but start differently far behind a boundary are summed in other orders: twice the bound of one."""
    g, M = _gen(30), 24
    x = torch.zeros(M, ld, device="cuda", dtype=TYPE[dtype])
    x[:, :D] = _randn(g, D).to(TYPE[dtype])
    y, _, _ = run_rms(lib, x, None, None, D, dtype, dtype, 0, pad=ld - D)
    one = y[:1].double()
    within(y, one.expand(M, D).to(TYPE[dtype]), one.abs() * 2 * (HALF[dtype] * 2 + 64 * U) + TINY[dtype])
    again, _, _ = run_rms(lib, x[:9], None, None, D, dtype, dtype, 0, pad=ld - D)
    assert torch.equal(again, y[:9])


# ------------------------------------------------------------------ rotary positions
def rope_ref(x, pos, freq, mscale, rot, inter, inverse):
    """x: (M, heads, hd) f64; returns (out, magnitude of the two terms) in f64."""
    a = pos.double()[:, None] * freq[None]
    c, s = (a.cos() * mscale)[:, None], (a.sin() * mscale * (-1 if inverse else 1))[:, None]
    i = torch.arange(rot // 2, device=x.device)
    p, q = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    out, mag = x.clone(), torch.zeros_like(x)
    out[..., p] = x[..., p] * c - x[..., q] * s
    out[..., q] = x[..., p] * s + x[..., q] * c
    mag[..., p] = mag[..., q] = (x[..., p].abs() + x[..., q].abs()) * abs(mscale)
    return out, mag


def rope_case(lib, M, heads, hd, rot, dtype, inter, inverse, pos_type=tb.F32, pos_stride=1, gap=0, hgap=0, span=366,
              mscale=1.0, planes=False, in_place=False, seed=0):
    """planes: heads outside, rows inside (head stride > row pitch)."""
    g = _gen(seed + M + 31 * hd + rot)
    hs = hd + hgap
    ld = heads * hs + gap
    if planes:
        ld, hs = hd + hgap, M * (hd + hgap) + gap
    n = (M - 1) * ld + (heads - 1) * hs + hd
    flat = _randn(g, n).to(TYPE[dtype])
    x = flat.as_strided((M, heads, hd), (ld, hs, 1))
    pos = torch.randint(0, span, (M, max(pos_stride, 1)), device="cuda", generator=g).to(TYPE[pos_type])
    p = pos[:, 0] if pos_stride else pos[:1, 0].expand(M)
    freq = torch.from_numpy(tb.rope_freqs(rot)[0]).cuda()
    want, mag = rope_ref(x.double(), p, freq, mscale, rot, inter, inverse)
    oflat = flat if in_place else torch.full((n,), 77.0, device="cuda").to(TYPE[dtype])
    before = oflat.clone()
    assert lib.tcb_op_rope(_p(flat), ld, hs, dtype, _p(pos), pos_stride, pos_type, _p(freq), mscale, rot, int(inter),
                           int(inverse), _p(oflat), ld, hs, M, heads, hd, _stream()) == 0
    torch.cuda.synchronize()
    out = oflat.as_strided((M, heads, hd), (ld, hs, 1))
    within(out, want.to(TYPE[dtype]), mag * 10 * U + want.abs() * 2 * HALF[dtype] + TINY[dtype])
    assert torch.equal(out[..., rot:].double(), want[..., rot:])
    out.copy_(before.as_strided(out.shape, out.stride()))
    assert torch.equal(oflat, before)  # nothing between the heads or rows was written


@pytest.mark.parametrize("dtype", [tb.BF16, tb.F16, tb.F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("M,heads,hd,rot", [(1, 1, 2, 2), (1, 8, 160, 160), (40, 8, 160, 160), (13, 3, 128, 64), (7, 5, 51, 26),
                                            (130, 10, 64, 16), (33, 2, 96, 90), (5, 1, 1024, 1024), (3, 48, 256, 130),
                                            (2, 3, 24, 8), (1000, 1, 16, 16)])
def test_rope(lib, M, heads, hd, rot, dtype, inter):
    rope_case(lib, M, heads, hd, rot, dtype, inter, False)
    rope_case(lib, M, heads, hd, rot, dtype, inter, True, mscale=1.25, gap=hd, hgap=8)
    rope_case(lib, M, heads, hd, rot, dtype, inter, False, in_place=True, gap=3, hgap=1)


@pytest.mark.parametrize("pos_type,stride", [(tb.F32, 1), (tb.F32, 3), (tb.F32, 11), (tb.F32, 0), (tb.I32, 1), (tb.I32, 2),
                                             (tb.I64, 1), (tb.I64, 0)])
def test_rope_positions(lib, pos_type, stride):
    rope_case(lib, 77, 4, 64, 64, tb.F32, False, False, pos_type=pos_type, pos_stride=stride, span=4_000_000)
    rope_case(lib, 77, 4, 64, 48, tb.BF16, True, False, pos_type=pos_type, pos_stride=stride, span=4_000_000)


@pytest.mark.parametrize("dtype", [tb.BF16, tb.F32])
def test_rope_head_planes(lib, dtype):
    """Heads outside the rows: (head, row, column) order, aligned and not."""
    rope_case(lib, 60, 6, 64, 64, dtype, False, False, planes=True)
    rope_case(lib, 61, 5, 66, 32, dtype, True, False, planes=True, gap=5, hgap=1)


def test_rope_far_positions(lib):
    """Positions past 2^32: the angle keeps its phase. f64 holds pos * freq to 2^-53 of it: 2^40 rad to 2^-13 rad on both
    sides, so positions stay below 2^33, where both agree to 2^-20 rad; the tolerance adds twice that."""
    pos = torch.tensor([2 ** 33 - 1, 2 ** 32 + 12345, -(2 ** 31) - 7, -1, 0], device="cuda")
    freq = torch.from_numpy(tb.rope_freqs(64)[0]).cuda()
    x = _randn(_gen(6), 5, 2, 64)
    out = torch.empty_like(x)
    assert lib.tcb_op_rope(_p(x), 128, 64, tb.F32, _p(pos), 1, tb.I64, _p(freq), 1.0, 64, 0, 0, _p(out), 128, 64, 5, 2, 64,
                           _stream()) == 0
    want, mag = rope_ref(x.double(), pos, freq, 1.0, 64, False, False)
    within(out, want, mag * (10 * U + 2.0 ** -19))


def test_rope_turns_back_and_gradient(lib):
    """inverse undoes the turn, and is the gradient: <turn(x), w> and <x, inverse(w)> are equal, also against differences."""
    g = _gen(8)
    M, H, hd, rot = 9, 3, 48, 32
    x, w, d = _randn(g, M, H * hd), _randn(g, M, H * hd), _randn(g, M, H * hd)
    pos = torch.arange(M, device="cuda", dtype=torch.int32) * 100
    freq = torch.from_numpy(tb.rope_freqs(rot)[0]).cuda()

    def turn(v, inverse):
        o = torch.empty_like(v)
        assert lib.tcb_op_rope(_p(v), H * hd, hd, tb.F32, _p(pos), 1, tb.I32, _p(freq), 1.5, rot, 1, inverse, _p(o), H * hd, hd,
                               M, H, hd, _stream()) == 0
        return o

    back = turn(turn(x, 0), 1).view(M, H, hd)
    want = x.view(M, H, hd).double().clone()
    want[..., :rot] *= 1.5 ** 2
    within(back, want, 2.25 * 40 * U * 2 * x.abs().max().item())
    grad = turn(w, 1).double()
    n = M * H * hd
    scale = (w.double().norm() * d.double().norm()).item() * 1.5
    lhs = (turn(d, 0).double() * w.double()).sum()  # the turn is linear: its difference along d
    assert abs((lhs - (grad * d.double()).sum()).item()) <= scale * 20 * U
    eps = 2.0 ** -8
    diff = (turn(x + eps * d, 0).double() - turn(x - eps * d, 0).double()) / (2 * eps)
    assert abs((diff * w.double()).sum().item() - (grad * d.double()).sum().item()) <= n ** 0.5 * scale * 20 * U / eps


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("dtype", [tb.BF16, tb.F32])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_shifted_pointers(lib, shift, dtype, inter):
    """x and out some elements behind a boundary; rotated parts that are and are not whole vectors of either layout."""
    g, M, H, hd = _gen(14), 11, 3, 64
    for rot in (8, 16, 24, 40, 64):
        buf = _randn(g, M * H * hd + 8).to(TYPE[dtype])
        out = torch.zeros_like(buf)
        x = buf[shift:shift + M * H * hd].view(M, H, hd)
        pos = torch.arange(M, device="cuda", dtype=torch.float32)
        freq = torch.from_numpy(tb.rope_freqs(rot)[0]).cuda()
        want, mag = rope_ref(x.double(), pos, freq, 1.0, rot, inter, False)
        assert lib.tcb_op_rope(buf[shift:].data_ptr(), H * hd, hd, dtype, _p(pos), 1, tb.F32, _p(freq), 1.0, rot, int(inter), 0,
                               out[shift:].data_ptr(), H * hd, hd, M, H, hd, _stream()) == 0
        within(out[shift:shift + M * H * hd].view(M, H, hd), want.to(TYPE[dtype]),
               mag * 10 * U + want.abs() * 2 * HALF[dtype] + TINY[dtype])
        assert not out[:shift].any() and not out[shift + M * H * hd:].any()


@pytest.mark.parametrize("dtype", [tb.BF16, tb.F16, tb.F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads,hd,rot", [(8, 151, 90), (1, 3, 2), (3, 51, 26), (19, 208, 82), (5, 66, 64), (40, 255, 254), (1, 1023, 6),
                                          (100, 257, 130)])
def test_rope_long_odd(lib, heads, hd, rot, dtype, inter):
    """Long streams of heads that no vector fits: packed, with columns behind the heads, in place, and in gaps."""
    rope_case(lib, 2500, heads, hd, rot, dtype, inter, False, span=366)
    rope_case(lib, 2049, heads, hd, rot, dtype, inter, True, gap=16 if heads < 50 else 0, pos_type=tb.I64, span=9999)
    rope_case(lib, 2049, heads, hd, rot, dtype, inter, False, gap=5, in_place=True)
    if heads < 50:
        rope_case(lib, 2050, heads, hd, rot, dtype, inter, False, hgap=1)


@pytest.mark.parametrize("shift", [0, 1, 3, 7])
def test_rope_long_odd_shifted(lib, shift):
    """The same with x and out that start off a boundary, alike and not."""
    g, M, H, hd, rot = _gen(19), 2100, 3, 37, 22
    for other in (shift, shift + 8, shift + 2):
        buf = _randn(g, M * H * hd + 16).to(torch.bfloat16)
        out = torch.zeros_like(buf)
        x = buf[shift:shift + M * H * hd].view(M, H, hd)
        pos = torch.arange(M, device="cuda", dtype=torch.int32)
        freq = torch.from_numpy(tb.rope_freqs(rot)[0]).cuda()
        want, mag = rope_ref(x.double(), pos, freq, 1.0, rot, False, False)
        assert lib.tcb_op_rope(buf[shift:].data_ptr(), H * hd, hd, tb.BF16, _p(pos), 1, tb.I32, _p(freq), 1.0, rot, 0, 0,
                               out[other:].data_ptr(), H * hd, hd, M, H, hd, _stream()) == 0
        within(out[other:other + M * H * hd].view(M, H, hd), want.to(torch.bfloat16),
               mag * 10 * U + want.abs() * 2.0 ** -7 + TINY[tb.BF16])
        assert not out[:other].any() and not out[other + M * H * hd:].any()


def test_rope_far_pitch(lib):
    ld = 1_300_000_008
    buf = torch.empty(2 * ld + 64, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, 2, 32), (ld, 32, 1))
    x.copy_(_randn(_gen(9), 3, 2, 32))
    pos = torch.tensor([1, 2, 3], device="cuda", dtype=torch.int32)
    freq = torch.from_numpy(tb.rope_freqs(32)[0]).cuda()
    want, mag = rope_ref(x.double(), pos, freq, 1.0, 32, False, False)
    assert lib.tcb_op_rope(_p(buf), ld, 32, tb.BF16, _p(pos), 1, tb.I32, _p(freq), 1.0, 32, 0, 0, _p(buf), ld, 32, 3, 2, 32,
                           _stream()) == 0
    within(x, want.to(torch.bfloat16), mag * 10 * U + want.abs() * 2.0 ** -7)


def test_rope_f32_error(lib):
    """f32 results in the root mean square, against cosines and sines rounded once from f64: what the fraction of a turn loses in
    f32 is put back by one more rounding of each. That doubles their variance; the products' roundings are about as large and
    stay: sqrt((2 + 1) / (1 + 1)) < 1.25."""
    g, M, H, hd = _gen(28), 20000, 4, 128
    x = _randn(g, M, H, hd)
    x[:, 0, 64:], x[:, 1, :64] = 0, 0
    pos = torch.randint(0, 4_000_000, (M,), device="cuda", generator=g, dtype=torch.int32)
    freq, out = torch.from_numpy(tb.rope_freqs(hd)[0]).cuda(), torch.empty_like(x)
    assert lib.tcb_op_rope(_p(x), H * hd, hd, tb.F32, _p(pos), 1, tb.I32, _p(freq), 1.0, hd, 0, 0, _p(out), H * hd, hd, M, H, hd,
                           _stream()) == 0
    want, mag = rope_ref(x.double(), pos, freq, 1.0, hd, False, False)
    a = pos.double()[:, None] * freq
    c, s, p, q = a.cos().float()[:, None], a.sin().float()[:, None], x[..., :64], x[..., 64:]
    once = torch.cat([p * c - q * s, p * s + q * c], -1)

    def rms(y):
        return ((y.double() - want) / mag).square().mean().sqrt().item()

    assert rms(out) <= 1.25 * rms(once)


# ------------------------------------------------------------------ 4-bit product
def w4_case(lib, M, N, K, group, xtype, otype, xgroup=0, relu=False, res=False, bias=True, pad=0, seed=0, in_place=False):
    g = _gen(seed + M + 3 * N + 5 * K)
    ng = -(-K // group)
    codes = torch.randint(-8, 8, (N, K), device="cuda", generator=g, dtype=torch.int8)
    scales = ((0.5 + torch.rand(N, ng, device="cuda", generator=g)) / K ** 0.5).to(torch.bfloat16)
    w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), group, scales.float().cpu().numpy())).cuda()
    wd = codes.double() * scales.double().repeat_interleave(group, 1)[:, :K]
    x = _randn(g, M, K + pad)
    xs = None
    if xtype in TOP:
        x = (x * TOP[xtype] / 4).clamp(-TOP[xtype], TOP[xtype])
        xs = 0.01 + torch.rand(M, -(-K // xgroup) if xgroup else 1, device="cuda", generator=g) / TOP[xtype]
    x = (x.round() if xtype == tb.I8 else x).to(TYPE[xtype])
    xd = x[:, :K].double()
    if xs is not None:
        xd = xd * (xs.double().repeat_interleave(xgroup, 1)[:, :K] if xgroup else xs.double())
    b = 0.1 * _randn(g, N) if bias else None
    y = torch.full((M + 1, N + pad), 77.0, device="cuda").to(TYPE[otype])
    r = _randn(g, M, N + pad).to(TYPE[otype]) if res else None
    if in_place:
        y[:M] = r
        r = y
    want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias:
        want, mag = want + b.double(), mag + b.double().abs()
    if relu:
        want = want.relu()
    if res:
        rd = r[:M, :N].double()
        want, mag = want + rd, mag + rd.abs()
    edge = y[:, N:].clone()
    assert lib.tcb_op_gemv_w4(_p(x), K + pad, xtype, _p(xs), xgroup, _p(w), group, _p(b), int(relu), _p(r), N + pad, _p(y),
                              N + pad, otype, M, N, K, _stream()) == 0
    torch.cuda.synchronize()
    tol = mag * (K + K / 16 + 16) * 2 * U + want.abs() * 2 * HALF[otype] + TINY[otype]
    within(y[:M, :N], want.to(TYPE[otype]), tol)
    assert torch.equal(y[:, N:], edge) and (y[M] == 77).all()
    # the bound grows with K; the typical error does not: 99% within a few roundings of the magnitudes' root
    err = (y[:M, :N].double() - want).abs()
    usual = (want.abs() * 2 * HALF[otype] + mag * 16 * U + TINY[otype])
    assert (err <= usual).double().mean().item() >= 0.99


W4_SIZES = [(1, 1, 1), (1, 16, 128), (1, 128, 2560), (2, 17, 129), (3, 100, 31), (8, 640, 640), (9, 48, 1000), (16, 33, 512),
            (17, 1920, 640), (1, 2560, 1280), (31, 65, 4096), (40, 130, 640), (64, 31, 300), (65, 64, 640), (130, 48, 256),
            (1, 7, 16385), (5, 16, 20000), (1, 5000, 128), (33, 4099, 250)]


@pytest.mark.parametrize("M,N,K", W4_SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_gemv_w4(lib, M, N, K, group):
    w4_case(lib, M, N, K, group, tb.BF16, tb.BF16)
    w4_case(lib, M, N, K, group, tb.F16, tb.F32, relu=True, pad=1)


@pytest.mark.parametrize("M,N,K", [(1, 48, 640), (4, 33, 1000), (13, 100, 250), (40, 1920, 640), (67, 17, 130)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xgroup", [0, 32, 64, 128])
@pytest.mark.parametrize("xtype", [tb.I8, tb.E4M3])
def test_gemv_w4_codes(lib, M, N, K, group, xgroup, xtype):
    w4_case(lib, M, N, K, group, xtype, tb.F32, xgroup=xgroup)
    w4_case(lib, M, N, K, group, xtype, tb.BF16, xgroup=xgroup, res=True, pad=3)


def test_gemv_w4_epilogues(lib):
    for otype in (tb.BF16, tb.F16, tb.F32):
        w4_case(lib, 5, 100, 640, 64, tb.BF16, otype, relu=True, res=True, bias=False)
        w4_case(lib, 5, 100, 640, 64, tb.F16, otype, res=True, in_place=True, pad=4)
        w4_case(lib, 20, 257, 384, 128, tb.F16, otype, bias=False)


def test_gemv_w4_largest(lib):
    w4_case(lib, 3, 16384, 8192, 128, tb.BF16, tb.BF16)
    w4_case(lib, 32, 4096, 16384, 64, tb.F16, tb.F16)


@pytest.mark.parametrize("M,N,K,xtype", [(1, 40, 65536, tb.BF16), (9, 17, 65500, tb.F16), (3, 33, 40000, tb.E4M3),
                                         (33, 20, 16384, tb.BF16), (32, 4096, 8192, tb.BF16), (29, 700, 10001, tb.F16),
                                         (17, 8191, 5001, tb.I8), (300, 70, 700, tb.BF16), (1, 60000, 128, tb.BF16),
                                         (5, 2000, 7000, tb.F16), (1, 256, 16384, tb.BF16),
                                         (70000, 20, 130, tb.F16)])
def test_gemv_w4_cuts(lib, M, N, K, xtype):
    """Sizes whose token rows or weight rows make the launch split K over clusters, slice a tile's records over warps, join in
    several batches, or cut the token rows."""
    for group in (32, 128):
        w4_case(lib, M, N, K, group, xtype, tb.F32, xgroup=64 if xtype == tb.E4M3 else 0, res=True, pad=1)
        w4_case(lib, M, N, K, group, xtype, tb.BF16, relu=True)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
@pytest.mark.parametrize("xtype", [tb.BF16, tb.I8])
def test_gemv_w4_shifted_x(lib, shift, xtype):
    """x some elements behind a boundary, with aligned and unaligned pitches."""
    g = _gen(15)
    codes = torch.randint(-8, 8, (50, 300), generator=torch.Generator().manual_seed(3), dtype=torch.int8)
    w = torch.from_numpy(tb.w4_pack(codes.numpy(), 64, np.ones((50, 5), np.float32))).cuda()
    for ld in (304, 301):
        buf = (20 * _randn(g, 6 * ld + 16)).round().to(TYPE[xtype])
        x = buf[shift:shift + 6 * ld].view(6, ld)[:, :300]
        xs = torch.full((6, 1), 0.5, device="cuda") if xtype == tb.I8 else None
        y = torch.zeros(6, 50, device="cuda")
        assert lib.tcb_op_gemv_w4(buf[shift:].data_ptr(), ld, xtype, _p(xs), 0, _p(w), 64, None, 0, None, 0, _p(y), 50, tb.F32,
                                  6, 50, 300, _stream()) == 0
        # whole numbers below 2^24 throughout: exact
        assert torch.equal(y.double(), x.double() @ codes.cuda().double().t() * (0.5 if xtype == tb.I8 else 1))


def test_gemv_w4_same_bits_wherever_x_starts(lib):
    g = _gen(21)
    for M, N, K in ((1, 500, 4000), (17, 3000, 10001), (30, 100, 16384)):
        codes = torch.randint(-8, 8, (N, K), generator=torch.Generator().manual_seed(4), dtype=torch.int8)
        w = torch.from_numpy(tb.w4_pack(codes.numpy(), 128, np.full((N, -(-K // 128)), 0.01, np.float32))).cuda()
        x0, ys = _randn(g, M, K).to(torch.bfloat16), []
        for ld, shift in ((-(-K // 8) * 8, 0), (K + 1, 0), (K, 3)):
            buf = torch.zeros(M * ld + 8, device="cuda", dtype=torch.bfloat16)
            x = buf[shift:shift + M * ld].view(M, ld)
            x[:, :K] = x0
            ys.append(torch.zeros(M, N, device="cuda"))
            assert lib.tcb_op_gemv_w4(buf[shift:].data_ptr(), ld, tb.BF16, None, 0, _p(w), 128, None, 0, None, 0, _p(ys[-1]), N,
                                      tb.F32, M, N, K, _stream()) == 0
        assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


@pytest.mark.parametrize("K", [1024, 2048])
def test_gemv_w4_most_weight_rows(lib, K):
    """2^24 weight rows with several tiles of 32 token rows: a cluster's sums for them all are 2^31 bytes. The weight rows
    repeat, so the outputs have to, bit for bit."""
    M, N, R = 320, 1 << 24, 64
    codes = np.random.default_rng(5).integers(-8, 8, (R, K), dtype=np.int8)
    w = torch.from_numpy(tb.w4_pack(codes, 128, np.full((R, K // 128), 0.0625, np.float32))).cuda().repeat(N // R)
    x = _randn(_gen(22), M, K).to(torch.bfloat16)
    y = torch.full((M, N), float("nan"), device="cuda", dtype=torch.bfloat16)
    assert lib.tcb_op_gemv_w4(_p(x), K, tb.BF16, None, 0, _p(w), 128, None, 0, None, 0, _p(y), N, tb.BF16, M, N, K, _stream()) == 0
    wd = torch.from_numpy(codes).cuda().double() * 0.0625
    want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    sums = mag * (K + K / 16 + 16) * 2 * U
    within(y[:, :R], want, sums + (want.abs() + sums) * HALF[tb.BF16] + TINY[tb.BF16])
    for row in y:
        assert torch.equal(row.view(-1, R), row[:R].expand(N // R, R))


def test_gemv_w4_far_values(lib):
    """bf16 token rows of any size: each group is scaled by its largest value, which costs what is 2^-31 of it and smaller at
    most 2^-39 of it; the tolerance adds that times the weights' magnitudes. Sums are held times 2^-12 while subnormal steps
    are 2^-149: four groups' roundings are 4 x 2^-150 x 2^12 < 2^-135."""
    g = _gen(16)
    K, N = 512, 64
    codes = torch.randint(-8, 8, (N, K), device="cuda", generator=g, dtype=torch.int8)
    w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), 128, np.full((N, 4), 0.125, np.float32))).cuda()
    x = _randn(g, 8, K)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] *= torch.exp(20 * _randn(g, K))
    x[3] = 0
    x[4, 128:256] = 0
    x[5] = 3e38 * torch.sign(x[5]) * (torch.arange(K, device="cuda") == 77)
    x[6] = 1e-40
    x[7] *= torch.where(torch.arange(K, device="cuda") % 2 == 0, 1e18, 1e-18)
    x = x.to(torch.bfloat16)
    y = torch.zeros(8, N, device="cuda")
    assert lib.tcb_op_gemv_w4(_p(x), K, tb.BF16, None, 0, _p(w), 128, None, 0, None, 0, _p(y), N, tb.F32, 8, N, K, _stream()) == 0
    wd = codes.double() * 0.125
    want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    tops = x.double().abs().view(8, 4, 128).amax(2).repeat_interleave(128, 1)
    within(y, want.to(torch.float32), mag * (K + K / 16 + 16) * 2 * U + (tops * 2.0 ** -39) @ wd.abs().t() + 2.0 ** -135)


def test_gemv_w4_infinite_results(lib):
    """An infinity times codes of one sign is that infinity, of both signs NaN, whatever slice or group it is in."""
    K, N = 2048, 20
    codes = np.ones((N, K), np.int8)
    codes[1] = -3
    codes[2, ::2] = -2
    codes[3, 5] = 0
    for at in (5, 1999):
        w = torch.from_numpy(tb.w4_pack(codes, 128, np.ones((N, 16), np.float32))).cuda()
        x = torch.ones(3, K, device="cuda")
        x[0, at] = float("inf")
        x[1, at] = float("-inf")
        x[2, at - 1] = x[2, at] = float("inf")
        for xtype in (tb.BF16, tb.F16):
            xt = x.to(TYPE[xtype])
            y = torch.zeros(3, N, device="cuda")
            assert lib.tcb_op_gemv_w4(_p(xt), K, xtype, None, 0, _p(w), 128, None, 0, None, 0, _p(y), N, tb.F32, 3, N, K,
                                      _stream()) == 0
            want = xt.double() @ torch.from_numpy(codes).cuda().double().t()
            assert torch.equal(torch.nan_to_num(y.double(), 7, 8, 9), torch.nan_to_num(want, 7, 8, 9))


def test_gemv_w4_nan_and_inf_stay_in_their_row(lib):
    """A NaN or an infinity in one token reaches that token's outputs only (a code of zero times infinity is NaN)."""
    g = _gen(2)
    x = _randn(g, 5, 256).to(torch.bfloat16)
    x[1, 3], x[3, 255] = float("nan"), float("inf")
    codes = torch.randint(1, 8, (32, 256), generator=torch.Generator().manual_seed(1), dtype=torch.int8)
    w = torch.from_numpy(tb.w4_pack(codes.numpy(), 64, np.ones((32, 4), np.float32))).cuda()
    y = torch.zeros(5, 32, device="cuda")
    assert lib.tcb_op_gemv_w4(_p(x), 256, tb.BF16, None, 0, _p(w), 64, None, 0, None, 0, _p(y), 32, tb.F32, 5, 32, 256,
                              _stream()) == 0
    assert torch.isnan(y[1]).all() and torch.isposinf(y[3]).all() and torch.isfinite(y[[0, 2, 4]]).all()


@pytest.mark.parametrize("K, group, xgroup", [(2045, 32, 64), (131, 128, 32), (7, 64, 0)])
def test_gemv_w4_infinity_in_the_last_column(lib, K, group, xgroup):
    """Rows that end inside a step of columns: an infinite last value, or an infinite last scale of 8-bit rows."""
    N, ng = 20, -(-K // group)
    codes = np.random.default_rng(6).integers(1, 8, (N, K), dtype=np.int8)
    codes[1, -1], codes[2, -1], codes[3] = 0, -3, -1
    w = torch.from_numpy(tb.w4_pack(codes, group, np.ones((N, ng), np.float32))).cuda()
    wd = torch.from_numpy(codes).cuda().double()

    def check(x, xtype, xs, xd):
        y = torch.zeros(2, N, device="cuda")
        assert lib.tcb_op_gemv_w4(_p(x), K, xtype, _p(xs), xgroup if xs is not None else 0, _p(w), group, None, 0, None, 0,
                                  _p(y), N, tb.F32, 2, N, K, _stream()) == 0
        assert torch.equal(torch.nan_to_num(y.double(), 7, 8, 9), torch.nan_to_num(xd @ wd.t(), 7, 8, 9))

    x = torch.ones(2, K, device="cuda")
    x[1, -1] = float("inf")
    for xtype in (tb.BF16, tb.F16):
        xt = x.to(TYPE[xtype])
        check(xt, xtype, None, xt.double())
    per = xgroup or K
    xs = torch.ones(2, -(-K // per), device="cuda")
    xs[1, -1] = float("inf")
    for xtype in (tb.I8, tb.E4M3):
        xt = torch.ones(2, K, device="cuda").to(TYPE[xtype])
        check(xt, xtype, xs, xt.double() * xs.double().repeat_interleave(per, 1)[:, :K])


@pytest.mark.parametrize("M,N,K", [(1, 40, 1024), (3, 2048, 8192), (20, 64, 1000), (40, 100, 257)])
@pytest.mark.parametrize("xtype,large,usual", [(tb.F16, 60000.0, 2e-3), (tb.F16, 1e3, 1e-3), (tb.BF16, 1e4, 1.0), (tb.BF16, 1e8, 1.0),
                                               (tb.BF16, 1e30, 1.0), (tb.I8, 127.0, 1.0), (tb.E4M3, 448.0, 2.0 ** -6)])
def test_gemv_w4_large_values_under_codes_of_zero(lib, M, N, K, xtype, large, usual):
    """A large activation adds nothing where the code is 0: the bound stays that of the other terms' magnitudes, each
    term and each sum rounded as elsewhere, and 99% of the results are within a few roundings."""
    g, cols = _gen(23), [5, K // 2, K - 1]
    for group, xgroup in ((128, 0), (32, 64)):
        codes = torch.randint(-1, 2, (N, K), device="cuda", generator=g, dtype=torch.int8)
        codes[::2, cols] = 0
        codes[1::2, cols] = 1
        w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), group, np.ones((N, -(-K // group)), np.float32))).cuda()
        x = usual * _randn(g, M, K)
        x[:, cols] = torch.tensor([large, -large, large], device="cuda")
        x, xs, per = (x.round() if xtype == tb.I8 else x).to(TYPE[xtype]), None, 0
        xd = x.double()
        if xtype in TOP:
            per = xgroup
            xs = 0.5 + torch.rand(M, -(-K // per) if per else 1, device="cuda", generator=g)
            xd = xd * (xs.double().repeat_interleave(per, 1)[:, :K] if per else xs.double())
        y = torch.zeros(M, N, device="cuda")
        assert lib.tcb_op_gemv_w4(_p(x), K, xtype, _p(xs), per, _p(w), group, None, 0, None, 0, _p(y), N, tb.F32, M, N, K,
                                  _stream()) == 0
        wd = codes.double()
        want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
        within(y, want, mag * (K + K / 16 + 16) * 2 * U + want.abs() * U)
        assert ((y.double() - want).abs() <= want.abs() * 2 * U + mag * 16 * U).double().mean().item() >= 0.99


@pytest.mark.parametrize("xtype", [tb.BF16, tb.F16, tb.I8, tb.E4M3])
def test_gemv_w4_codes_of_zero(lib, xtype):
    """All codes 0 under scales that are not: bias and residual and nothing else."""
    g, N = _gen(24), 100
    for M, K in ((1, 8192), (7, 700), (33, 2000)):
        codes, ng = np.zeros((N, K), np.int8), -(-K // 64)
        w = torch.from_numpy(tb.w4_pack(codes, 64, np.full((N, ng), 3.0, np.float32))).cuda()
        x = 10 * _randn(g, M, K)
        x = (x.round() if xtype == tb.I8 else x).to(TYPE[xtype])
        xs = 0.5 + torch.rand(M, ng, device="cuda", generator=g) if xtype in TOP else None
        b, r = _randn(g, N), _randn(g, M, N)
        for bias, res in ((None, None), (b, r)):
            y = torch.full((M, N), 77.0, device="cuda")
            assert lib.tcb_op_gemv_w4(_p(x), K, xtype, _p(xs), 64 if xtype in TOP else 0, _p(w), 64, _p(bias), 0, _p(res), N, _p(y),
                                      N, tb.F32, M, N, K, _stream()) == 0
            assert torch.equal(y, torch.zeros(M, N, device="cuda") if bias is None else r + b)


@pytest.mark.parametrize("xgroup", [0, 32, 64, 128])
@pytest.mark.parametrize("xtype", [tb.I8, tb.E4M3])
@pytest.mark.parametrize("xscale,wscale", [(2.0 ** 117, 2.0 ** -20), (2.0 ** 124, 2.0 ** -40), (2.0 ** -110, 2.0 ** 120), (2.0 ** 100, 2.0 ** 60)])
def test_gemv_w4_far_scales(lib, xtype, xgroup, xscale, wscale):
    """Finite scales of 8-bit rows, however far from 1: an output is finite where its sum is, and infinite where that is past
    f32's end. A row of another scale beside them stays within the same bound."""
    for M, N, K, group in ((3, 40, 384, 128), (9, 70, 4100, 32)):
        g, nxg, ng = _gen(25), -(-K // xgroup) if xgroup else 1, -(-K // group)
        codes = torch.randint(-8, 8, (N, K), device="cuda", generator=g, dtype=torch.int8)
        codes[:4] = 7
        w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), group, np.full((N, ng), wscale, np.float32))).cuda()
        x = TOP[xtype] * (1 - torch.rand(M, K, device="cuda", generator=g))
        x[0, ::3] *= -1
        x = (x.floor() if xtype == tb.I8 else x).to(TYPE[xtype])
        xs = xscale * (1 - 0.5 * torch.rand(M, nxg, device="cuda", generator=g))
        xs[2] = 0.5
        y = torch.zeros(M, N, device="cuda")
        assert lib.tcb_op_gemv_w4(_p(x), K, xtype, _p(xs), xgroup, _p(w), group, None, 0, None, 0, _p(y), N, tb.F32, M, N, K,
                                  _stream()) == 0
        xd = x.double() * xs.double().repeat_interleave(xgroup or K, 1)[:, :K]
        wd = codes.double() * wscale
        want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
        finite = mag < 2.0 ** 127
        assert finite[:2].all() if xscale * wscale < 1e30 else (want[1].abs() > 2.0 ** 129).all()
        within(y, want.to(torch.float32), mag * (K + K / 16 + 16) * 2 * U + want.abs() * U)


@pytest.mark.parametrize("xgroup", [0, 32, 128])
@pytest.mark.parametrize("xtype", [tb.I8, tb.E4M3])
def test_gemv_w4_8_bit_rows_that_are_not_finite(lib, xtype, xgroup):
    """Rows with a NaN code or scale are NaN; under an infinite scale each product has its sign (0 times it is NaN); other rows
    stay as they are. The weights' zeros and signs differ from output to output."""
    M, N, K = 12, 150, 2300
    g, nxg = _gen(29), -(-K // xgroup) if xgroup else 1
    codes = torch.randint(-8, 8, (N, K), device="cuda", generator=g, dtype=torch.int8)
    codes[::3] = 1 + codes[::3].abs() % 7  # one sign, no zeros
    codes[1::3, 2200:] = -3
    w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), 64, np.full((N, 36), 0.25, np.float32))).cuda()
    x = torch.randint(1, 9, (M, K), device="cuda", generator=g).float()
    x[5] *= torch.where(torch.rand(K, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    x[6, K - 1], x[9, 40:50] = 0, 0
    x = x.to(TYPE[xtype])
    xs = torch.full((M, nxg), 0.5, device="cuda")
    xs[1], xs[2, -1], xs[9, 0] = float("nan"), float("nan"), float("inf")
    xs[4, -1], xs[5], xs[6, -1], xs[7] = float("inf"), float("-inf"), float("inf"), float("-inf")
    if xtype == tb.E4M3:
        x.view(torch.uint8)[8, 1777], x.view(torch.uint8)[10] = 0x7f, 0xff
    y = torch.zeros(M, N, device="cuda")
    assert lib.tcb_op_gemv_w4(_p(x), K, xtype, _p(xs), xgroup, _p(w), 64, None, 0, None, 0, _p(y), N, tb.F32, M, N, K, _stream()) == 0
    xd = x.double() * xs.double().repeat_interleave(xgroup or K, 1)[:, :K]
    # the library's product in 64 bits may skip zeros: one sum of products per output
    want = torch.stack([(row * codes.double() * 0.25).sum(1) for row in xd])
    assert torch.equal(torch.nan_to_num(y.double(), 7, 8, 9), torch.nan_to_num(want, 7, 8, 9))  # whole quarters below 2^24: exact


# ------------------------------------------------------------------ together
def test_zero_rows_are_a_no_op(lib):
    x = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    assert lib.tcb_op_rmsnorm(None, 64, None, 0, None, 0, None, 1e-6, tb.BF16, None, 64, tb.BF16, None, 0, 0, 64, _stream()) == 0
    assert lib.tcb_op_rope(None, 64, 32, tb.BF16, None, 1, tb.F32, None, 1.0, 32, 0, 0, None, 64, 32, 0, 2, 32, _stream()) == 0
    assert lib.tcb_op_gemv_w4(None, 64, tb.BF16, None, 0, None, 64, None, 0, None, 0, None, 8, tb.BF16, 0, 8, 64, _stream()) == 0
    torch.cuda.synchronize()
    assert (x == 1).all()


class Block:
    """The front of a pre-norm block on one packed stream: h = x + res, n = norm(h) in 8 bits, qkv = W4 n, q and k turned in
    place by the records' day of year, attention over series of T tokens."""

    def __init__(self, P, T, seed, code=tb.E4M3):
        g = _gen(seed)
        self.P, self.T, self.M, self.code = P, T, P * T, code
        M = self.M
        self.x, self.res = _randn(g, M, 640).to(torch.bfloat16), _randn(g, M, 640).to(torch.bfloat16)
        self.g = 1 + 0.1 * _randn(g, 640)
        self.rec = torch.randint(1, 367, (M, 11), device="cuda", generator=g).float()
        self.freq = torch.from_numpy(tb.rope_freqs(160)[0]).cuda()
        self.wf = (_randn(g, 1920, 640) / 640 ** 0.5).cpu().numpy()
        self.w = torch.from_numpy(tb.w4_pack(self.wf, 64)).cuda()
        self.bias = 0.1 * _randn(g, 1920)
        self.h = torch.zeros_like(self.x)
        self.n = torch.zeros(M, 640, device="cuda", dtype=TYPE[code])
        self.s = torch.zeros(M, 5, device="cuda")
        self.qkv = torch.zeros(M, 1920, device="cuda", dtype=torch.bfloat16)
        self.before = torch.zeros_like(self.qkv)
        self.att = torch.zeros_like(self.x)

    def run(self, lib, stream=None):
        st = stream or _stream()
        M = self.M
        assert lib.tcb_op_rmsnorm(_p(self.x), 640, _p(self.res), 640, _p(self.h), 640, _p(self.g), 1e-6, tb.BF16, _p(self.n),
                                  640, self.code, _p(self.s), 128, M, 640, st) == 0
        for out in (self.qkv, self.before):
            assert lib.tcb_op_gemv_w4(_p(self.n), 640, self.code, _p(self.s), 128, _p(self.w), 64, _p(self.bias), 0, None, 0,
                                      _p(out), 1920, tb.BF16, M, 1920, 640, st) == 0
        assert lib.tcb_op_rope(_p(self.qkv), 1920, 160, tb.BF16, self.rec.data_ptr() + 40, 11, tb.F32, _p(self.freq), 1.0, 160, 0,
                               0, _p(self.qkv), 1920, 160, M, 8, 160, st) == 0
        assert lib.tcb_op_attention(_p(self.qkv), None, self.T, self.P, self.T, _p(self.att), st) == 0

    def check(self):
        from test_gpu_ops import attention_ref, close_bf16
        from test_token_ops import unpack
        h, v = rms_ref(self.x, self.res, self.g, 1e-6)
        assert torch.equal(self.h, h)
        check_rms(h, v, self.n, self.code, 128, self.s)
        q, s = unpack(self.w.cpu().numpy(), 1920, 640, 64)
        wd = torch.from_numpy(q * np.repeat(s, 64, 1).astype(np.float64)).cuda()
        xd = self.n.double() * self.s.double().repeat_interleave(128, 1)
        want, mag = xd @ wd.t() + self.bias.double(), xd.abs() @ wd.abs().t() + self.bias.double().abs()
        within(self.before, want.to(torch.bfloat16), mag * 700 * 2 * U + want.abs() * 2.0 ** -7)
        # against the weights before quantisation: 4 bits move a product's sum by its own rounding, at most half a scale
        # (max|w| / 14 of a group) per term
        assert ((want - xd @ torch.from_numpy(self.wf).cuda().double().t() - self.bias.double()).abs()
                <= xd.abs() @ torch.from_numpy(np.repeat(s, 64, 1) * 0.54).cuda().double().t()).all()
        M = self.M
        turned, mag = rope_ref(self.before[:, :1280].double().view(M, 8, 160), self.rec[:, 10], self.freq, 1.0, 160, False, False)
        within(self.qkv[:, :1280].view(M, 8, 160), turned.to(torch.bfloat16), mag * 10 * U + turned.abs() * 2.0 ** -7)
        assert torch.equal(self.qkv[:, 1280:], self.before[:, 1280:])
        close_bf16(self.att, attention_ref(self.qkv, np.arange(self.P + 1) * self.T), ulps=3, atol=1e-2)


@pytest.mark.parametrize("P,T,code", [(1, 1, tb.E4M3), (1, 40, tb.E4M3), (3, 8, tb.I8), (1, 120, tb.I8)])
def test_block_front(lib, P, T, code):
    b = Block(P, T, P + T, code)
    b.run(lib)
    torch.cuda.synchronize()
    b.check()


def test_block_front_captured_and_replayed(lib):
    """Captured once, replayed on new inputs in the same buffers, while another block runs on a second stream."""
    a, b = Block(2, 16, 1), Block(2, 16, 2)
    a.run(lib)  # the attention kernels' first use sets their attributes
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        a.run(lib)
    fresh = Block(2, 16, 3)
    for name in ("x", "res", "rec"):
        getattr(a, name).copy_(getattr(fresh, name))
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            b.run(lib)
    torch.cuda.synchronize()
    a.check()
    b.check()


def test_captured_first_and_replayed(lib):
    """A size that splits K over clusters, whose kernel's first call on the device is the captured one, replayed on other
    inputs, and a second graph of the same sizes replayed between."""
    M, N, K, group = 25, 400, 9000, 64
    g, jobs = _gen(18), []
    for _ in range(2):
        codes = torch.randint(-8, 8, (N, K), device="cuda", generator=g, dtype=torch.int8)
        w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), group, np.full((N, -(-K // group)), 0.125, np.float32))).cuda()
        x, y = torch.zeros(M, K, device="cuda", dtype=torch.float16), torch.zeros(M, N, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert lib.tcb_op_gemv_w4(_p(x), K, tb.F16, None, 0, _p(w), group, None, 0, None, 0, _p(y), N, tb.F32, M, N, K,
                                      _stream()) == 0
        jobs.append((graph, codes.double() * 0.125, x, y, w))  # w: the graph reads it
    for _ in range(3):
        for graph, _, x, _, _ in jobs:
            x.copy_(_randn(g, M, K))
            graph.replay()
        for _, wd, x, y, _ in jobs:
            want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
            within(y, want, mag * (K + K / 16 + 16) * 2 * U + want.abs() * U)


def test_two_streams_at_once(lib):
    """The same operators on two streams that overlap, on sizes that split K over clusters."""
    g = _gen(17)
    jobs, M, N, K = [], 17, 2000, 10000
    for _ in range(2):
        codes = torch.randint(-8, 8, (N, K), device="cuda", generator=g, dtype=torch.int8)
        w = torch.from_numpy(tb.w4_pack(codes.cpu().numpy(), 128, np.full((N, -(-K // 128)), 0.125, np.float32))).cuda()
        jobs.append((torch.cuda.Stream(), w, _randn(g, M, K).to(torch.float16), torch.zeros(M, N, device="cuda")))
    torch.cuda.synchronize()

    def call(st, w, x, y):
        assert lib.tcb_op_gemv_w4(_p(x), K, tb.F16, None, 0, _p(w), 128, None, 0, None, 0, _p(y), N, tb.F32, M, N, K,
                                  st.cuda_stream) == 0

    for j in jobs:
        call(*j)
    torch.cuda.synchronize()
    alone = [j[3].clone() for j in jobs]
    for j in jobs:
        j[3].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for j in jobs:
            call(*j)
    torch.cuda.synchronize()
    for j, want in zip(jobs, alone):
        assert torch.equal(j[3], want)


def test_repeated_calls_give_the_same_bits(lib):
    a = Block(1, 64, 5)
    a.run(lib)
    first = [t.clone() for t in (a.h, a.n.view(torch.int8), a.s, a.qkv, a.att)]
    for _ in range(3):
        a.run(lib)
        for u, v in zip(first, (a.h, a.n.view(torch.int8), a.s, a.qkv, a.att)):
            assert torch.equal(u, v)
