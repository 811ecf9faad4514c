"""CPU tests of the token-stream operators (tcb_op_rmsnorm, tcb_op_rope,
tcb_op_gemv_w4): refused calls, the rotary frequencies and the packed form of
4-bit weights. Every refusal comes before any CUDA call, so none needs a GPU."""
import ctypes as C
import math

import numpy as np
import pytest

import tessera_b200 as tb

P = 0x1000  # a pointer that no refused call reads


def _rms(lib, **kw):
    a = dict(x=P, ldx=64, res=P, ldr=64, sum=P, lds=64, g=P, eps=1e-6, dtype=tb.BF16, y=P, ldy=64, ytype=tb.I8, scales=P,
             group=0, M=4, D=64, stream=None)
    assert set(kw) <= set(a)
    return lib.tcb_op_rmsnorm(*{**a, **kw}.values())


def _rope(lib, **kw):
    a = dict(x=P, ldx=128, hsx=32, dtype=tb.BF16, pos=P, pos_stride=1, pos_type=tb.F32, freq=P, mscale=1.0, rot=32,
             interleaved=0, inverse=0, out=2 * P, ldo=128, hso=32, M=4, heads=4, hd=32, stream=None)
    assert set(kw) <= set(a)
    return lib.tcb_op_rope(*{**a, **kw}.values())


def _w4(lib, **kw):
    a = dict(x=P, ldx=256, xtype=tb.E4M3, xscales=P, xgroup=0, w=P, group=64, bias=P, relu=0, res=P, ldr=48, out=2 * P,
             ldo=48, otype=tb.BF16, M=4, N=48, K=256, stream=None)
    assert set(kw) <= set(a)
    return lib.tcb_op_gemv_w4(*{**a, **kw}.values())


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=tb.I8), "dtype"), (dict(dtype=-1), "dtype"), (dict(dtype=tb.I64), "dtype"),
    (dict(ytype=tb.F16), "ytype"), (dict(ytype=7), "ytype"), (dict(M=-1), "M is negative"), (dict(D=0), "D is not"),
    (dict(D=16385, ldx=16385, ldr=16385, lds=16385, ldy=16385), "D is not"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(group=16), "group is not"),
    (dict(group=-32), "group is not"), (dict(ytype=tb.BF16, scales=None, group=32), "group without"),
    (dict(ytype=tb.BF16), "scales without"), (dict(scales=None), "scales is NULL"), (dict(ldx=63), "pitch"),
    (dict(ldr=63), "pitch"), (dict(lds=63), "pitch"), (dict(ldy=63), "pitch"), (dict(res=None), "sum without res"),
    (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(res=P + 1), "aligned"),
    (dict(sum=P + 1), "aligned"), (dict(g=P + 2), "aligned"), (dict(scales=P + 2), "aligned"),
    (dict(dtype=tb.F32, x=P + 2), "aligned"), (dict(ytype=tb.BF16, scales=None, y=P + 1), "aligned"),
    (dict(lds=72, y=2 * P), "another pitch"), (dict(ytype=tb.BF16, scales=None, y=3 * P, x=3 * P, ldy=80), "another pitch"),
    (dict(), "8-bit output over"), (dict(ytype=tb.BF16, scales=None, y=4 * P, res=4 * P, sum=5 * P), "y is res"),
])
def test_rmsnorm_refusals(kw, says, capfd):
    assert _rms(tb.load_library(), **kw) == -1
    err = capfd.readouterr().err
    assert err.startswith("tcb_op_rmsnorm: ") and says in err


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=tb.E4M3), "dtype"), (dict(pos_type=tb.BF16), "pos_type"), (dict(M=-1), "M is negative"),
    (dict(heads=0), "heads"), (dict(heads=65536), "heads"), (dict(hd=1), "hd is not"),
    (dict(hd=1025, hsx=1025, hso=1025), "hd is not"), (dict(rot=0), "rot"), (dict(rot=31), "rot"), (dict(rot=34), "rot"),
    (dict(hsx=31), "head stride"), (dict(hso=31), "head stride"), (dict(pos_stride=-1), "pos_stride"),
    (dict(ldx=-1), "pitch"), (dict(ldo=-128), "pitch"), (dict(ldo=127), "overlap"), (dict(ldo=0), "overlap"),
    (dict(ldo=32, hso=127), "overlap"), (dict(x=None), "NULL"), (dict(pos=None), "NULL"), (dict(freq=None), "NULL"),
    (dict(out=None), "NULL"), (dict(x=P + 1), "aligned"), (dict(out=2 * P + 1), "aligned"), (dict(pos=P + 2), "aligned"),
    (dict(pos_type=tb.I64, pos=P + 4), "aligned"), (dict(freq=P + 4), "aligned"),
    (dict(ldo=2 ** 62, hso=2 ** 62, M=2 ** 40, hd=32), "overlap"), (dict(out=P, ldx=130), "other strides"), (dict(out=P, hsx=33, ldx=132, ldo=132), "other strides"),
])
def test_rope_refusals(kw, says, capfd):
    assert _rope(tb.load_library(), **kw) == -1
    err = capfd.readouterr().err
    assert err.startswith("tcb_op_rope: ") and says in err


@pytest.mark.parametrize("kw,says", [
    (dict(xtype=tb.F32), "xtype"), (dict(xtype=tb.I32), "xtype"), (dict(otype=tb.E4M3), "otype"), (dict(M=-1), "M is not"), (dict(M=2 ** 18 + 1), "M is not"),
    (dict(N=0), "N is not"), (dict(K=0), "K not"), (dict(K=65537, ldx=65537), "K not"),
    (dict(group=16), "group"), (dict(group=0), "group"), (dict(xgroup=16), "xgroup"),
    (dict(xtype=tb.BF16, xscales=None, xgroup=32), "xgroup without"), (dict(xtype=tb.BF16), "xscales without"),
    (dict(xscales=None), "xscales is NULL"), (dict(ldx=255), "pitch"), (dict(ldo=47), "pitch"), (dict(ldr=47), "pitch"),
    (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(out=None), "NULL"), (dict(w=P + 8), "aligned"),
    (dict(res=2 * P, ldr=49), "another pitch"), (dict(N=2 ** 24 + 1, ldo=2 ** 25, ldr=2 ** 25), "N is not"),
    (dict(xtype=tb.BF16, xscales=None, x=P + 1), "aligned"), (dict(xscales=P + 2), "aligned"), (dict(bias=P + 2), "aligned"),
    (dict(res=P + 1), "aligned"), (dict(out=2 * P + 1), "aligned"), (dict(out=P, res=None), "out is x"),
])
def test_gemv_w4_refusals(kw, says, capfd):
    assert _w4(tb.load_library(), **kw) == -1
    err = capfd.readouterr().err
    assert err.startswith("tcb_op_gemv_w4: ") and says in err


def test_rope_freqs_formulas():
    """Each scaling against its formula in numpy f64 (pow may differ by a few ulp of f64)."""
    rot, base = 64, 10000.0
    f0 = base ** (-np.arange(0, rot, 2) / rot)
    f, m = tb.rope_freqs(rot)
    np.testing.assert_allclose(f, f0, rtol=1e-14)
    assert m == 1.0
    f, m = tb.rope_freqs(rot, base, tb.ROPE_LINEAR, 8.0)
    np.testing.assert_allclose(f, f0 / 8, rtol=1e-14)
    assert m == 1.0
    f, m = tb.rope_freqs(rot, base, tb.ROPE_BASE, 8.0)
    assert f[0] == 1.0 and m == 1.0
    np.testing.assert_allclose(f[-1], f0[-1] / 8, rtol=1e-13)  # the slowest pair slows by the factor
    f, m = tb.rope_freqs(rot, base, tb.ROPE_WAVES, 32.0, 8192.0, 32.0, 1.0)
    turns = 8192 * f0 / (2 * np.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    np.testing.assert_allclose(f, f0 * keep + f0 / 32 * (1 - keep), rtol=1e-14)
    assert keep[0] == 1 and keep[-1] == 0 and ((keep > 0) & (keep < 1)).any()
    assert m == np.float32(0.1 * math.log(32) + 1)
    # a factor of one leaves every frequency as it is
    for how in (tb.ROPE_LINEAR, tb.ROPE_BASE, tb.ROPE_WAVES):
        f, m = tb.rope_freqs(rot, base, how, 1.0, 8192.0)
        np.testing.assert_allclose(f, f0, rtol=1e-14)
        assert m == 1.0


@pytest.mark.parametrize("args", [
    (0, 1e4, 0, 1.0, 0.0, 0.0, 0.0), (3, 1e4, 0, 1.0, 0.0, 0.0, 0.0), (1026, 1e4, 0, 1.0, 0.0, 0.0, 0.0),
    (8, 1.0, 0, 1.0, 0.0, 0.0, 0.0), (8, math.nan, 0, 1.0, 0.0, 0.0, 0.0), (8, 1e4, 4, 1.0, 0.0, 0.0, 0.0),
    (8, 1e4, -1, 1.0, 0.0, 0.0, 0.0), (8, 1e4, 1, 0.5, 0.0, 0.0, 0.0), (8, 1e4, 1, math.inf, 0.0, 0.0, 0.0),
    (2, 1e4, 2, 2.0, 0.0, 0.0, 0.0), (8, 1e4, 3, 2.0, 0.0, 32.0, 1.0), (8, 1e4, 3, 2.0, 64.0, 1.0, 1.0),
    (8, 1e4, 3, 2.0, 64.0, 1.0, -1.0),
])
def test_rope_freqs_refusals(args, capfd):
    f = np.zeros(1024)
    m = C.c_float()
    assert tb.load_library().tcb_rope_freqs(*args, tb._ptr(f), C.byref(m)) == -1
    assert capfd.readouterr().err.startswith("tcb_rope_freqs: ")


def unpack(packed: np.ndarray, N: int, K: int, group: int):
    """The padded codes and scales of a packed matrix, read by the documented layout one element at a time."""
    per = 128 // group
    rec = 1024 + per * 32
    tiles, recs = -(-N // 16), -(-K // 128)
    p = packed.reshape(tiles, recs, rec)
    q = np.zeros((tiles * 16, recs * 128), np.int32)
    for r in range(16):
        for j in range(128):
            i, t, c = j // 32, j // 8 % 4, j % 8
            word = p[:, :, 512 * (r // 8) + 64 * (r % 8) + 16 * t + 4 * i:][:, :, :4].copy().view("<u4")[:, :, 0]
            nibble = c // 2 + 4 * (c % 2)
            q[r::16, j::128] = (word >> np.uint32(4 * nibble) & 15).astype(np.int32) - 8
    s = (p[:, :, 1024:].copy().view("<u2").astype(np.uint32) << 16).view(np.float32)
    s = s.reshape(tiles, recs, per, 16).transpose(0, 3, 1, 2).reshape(tiles * 16, recs * per)
    return q, s


@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (16, 128, 128), (17, 129, 64), (33, 250, 32), (48, 640, 128), (5, 97, 64)])
def test_w4_pack_codes_layout(N, K, group):
    rng = np.random.default_rng(N * K)
    codes = rng.integers(-8, 8, (N, K)).astype(np.int8)
    ng = -(-K // group)
    scales = rng.uniform(0.5, 2, (N, ng)).astype(np.float32)
    assert tb.load_library().tcb_w4_bytes(N, K, group) == -(-N // 16) * -(-K // 128) * (1024 + 4096 // group)
    q, s = unpack(tb.w4_pack(codes, group, scales), N, K, group)
    np.testing.assert_array_equal(q[:N, :K], codes)
    assert not q[N:].any() and not q[:, K:].any() and not s[N:].any() and not s[:, ng:].any()
    # scales are rounded to bf16, to nearest
    assert (np.abs(s[:N, :ng] - scales) <= scales * 2.0 ** -8).all()
    assert not (s[:N, :ng].view(np.uint32) & 0xFFFF).any()


@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (20, 300, 64), (16, 256, 128)])
def test_w4_pack_quantises(N, K, group):
    """Codes are the nearest multiple of the stored scale: off by at most half a scale, plus what the scale's own
    rounding (2^-8) moves the end of the range: 7 codes x 2^-8 of a scale."""
    rng = np.random.default_rng(7)
    w = rng.normal(size=(N, K)).astype(np.float32)
    w[0, :min(K, group)] = 0  # a group of zeros: scale 0, codes 0
    q, s = unpack(tb.w4_pack(w, group), N, K, group)
    q, s = q[:N, :K], np.repeat(s[:N], group, 1)[:, :K]
    assert np.abs(q).max() <= 7
    assert (np.abs(q * s - w) <= s * (0.5 + 7 * 2.0 ** -8) + 1e-30).all()
    assert not q[0, :min(K, group)].any() and not s[0, :min(K, group)].any()


def test_w4_pack_refusals(capfd):
    lib = tb.load_library()
    for bad in ((0, 128, 32), (16, 0, 32), (16, 128, 16), (16, 65537, 32), (-1, 128, 32), (2 ** 24 + 1, 128, 32)):
        assert lib.tcb_w4_bytes(*bad) == -1
        assert lib.tcb_w4_pack(P, *bad, P) == -1
        assert lib.tcb_w4_pack_codes(P, P, *bad, P) == -1
    out = np.zeros(lib.tcb_w4_bytes(1, 4, 32), np.uint8)
    codes, s = np.array([[0, 8, 0, 0]], np.int8), np.ones((1, 1), np.float32)
    assert lib.tcb_w4_pack_codes(tb._ptr(codes), tb._ptr(s), 1, 4, 32, tb._ptr(out)) == -1
    assert "-8..7" in capfd.readouterr().err
    codes[0, 1] = 7
    for v in (np.nan, np.inf, 3.4e38):  # the last one rounds to an infinite bf16
        s[0, 0] = v
        assert lib.tcb_w4_pack_codes(tb._ptr(codes), tb._ptr(s), 1, 4, 32, tb._ptr(out)) == -1
        assert "not finite" in capfd.readouterr().err
    for v, says in ((np.nan, "not finite"), (np.inf, "not finite")):
        w = np.array([[0, v, 0, 0]], np.float32)
        assert lib.tcb_w4_pack(tb._ptr(w), 1, 4, 32, tb._ptr(out)) == -1
        assert says in capfd.readouterr().err
    assert lib.tcb_w4_pack(None, 1, 4, 32, tb._ptr(out)) == -1
    assert lib.tcb_w4_pack_codes(tb._ptr(codes), None, 1, 4, 32, tb._ptr(out)) == -1
    with pytest.raises(ValueError):
        tb.w4_pack(codes, 32, np.ones((1, 2), np.float32))


@pytest.mark.parametrize("bad", [np.array([[0, 264, 0, 0]]), np.array([[0, -249, 0, 0]], np.int16), np.array([[0, 256, 0, 0]], np.uint16),
                                 np.array([[0, 1.5, 0, 0]]), np.array([[0, np.nan, 0, 0]]), np.array([[0, 8, 0, 0]])])
def test_w4_pack_codes_of_wider_types(bad):
    """Codes that no int8 holds are refused and not wrapped into the range; whole ones in range are taken from any type."""
    s = np.ones((1, 1), np.float32)
    with pytest.raises(ValueError):
        tb.w4_pack(bad, 32, s)
    good = np.array([[-8, 7, 0, 3]])
    want = tb.w4_pack(good.astype(np.int8), 32, s)
    for t in (np.int64, np.int16, np.float32):
        np.testing.assert_array_equal(tb.w4_pack(good.astype(t), 32, s), want)
