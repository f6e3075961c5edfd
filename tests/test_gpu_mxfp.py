"""Microscaled formats on the GPU: rounding and reading back bit for bit, the norm whose result is MXFP8, and the products over MXFP4
weights against 64 bits.

Tolerance of the products: elements multiply exactly (4 by 2 significant bits), so only sums round. An element's product meets at
most 128 additions inside a matrix instruction, one for each of the K/128 instructions, and one for each of up to 64 parts, terms or
wavefronts whose sums are joined: |error| <= (128 + K/128 + 64) 2^-24 sum |a w|. The f32 row of the decode product
is carried to 2^-38 of its block's largest, which is below one of those roundings per element for a spread of up to 2^14.
"""
import ctypes as C

import numpy as np
import pytest

import mx_oracle as mx

pytestmark = pytest.mark.gpu
EPS = 1e-6


def rng(*key):
    return np.random.default_rng(list(key))


def activations(r, rows, k):
    """Rows with some columns an order larger, some blocks of zeros, some of small numbers."""
    x = r.standard_normal((rows, k)) * np.where(r.random(k) < 0.02, 13, 1)
    b = x.reshape(rows, -1, 32)
    b[r.random(b.shape[:2]) < 0.02] = 0
    b[r.random(b.shape[:2]) < 0.02] *= 1e-4
    return x.astype(np.float32)


def weight(r, n, k):
    codes, scales = mx.quantize((r.standard_normal((n, k)) * 0.02).astype(np.float32), True)
    return codes, scales


def rows8(r, m, k):
    return mx.quantize(activations(r, m, k), False)


def guarded(lib, nbytes):
    """Room for nbytes with 256 bytes of 0xa5 behind them."""
    b = lib.empty_bytes(nbytes + 256)
    b.upload(np.full(nbytes + 256, 0xa5, np.uint8))
    return b


def taken(b, nbytes, dtype, shape):
    raw = b.numpy(np.uint8)
    assert (raw[nbytes:] == 0xa5).all(), "wrote behind the result"
    return raw[:nbytes].view(dtype).reshape(shape)


def half_types(x, t):
    if t == "f32":
        return x
    if t == "f16":
        return x.astype(np.float16)
    u = x.astype(np.float32).view(np.uint32)
    return ((u + 0x7fff + (u >> 16 & 1)) >> 16).astype(np.uint16)


def widened(x, t):
    return x.astype(np.float32) if t != "bf16" else (x.astype(np.uint32) << 16).view(np.float32)


def hard_values(r, rows, k):
    """What rounding can go wrong at: borders between codes, both neighbours of them, the block's largest below and above a power
    of two, subnormal blocks, zeros of both signs, infinities and NaN."""
    x = r.standard_normal((rows, k)).astype(np.float32)
    b = x.reshape(-1, 32)
    for i in range(len(b)):
        kind = i % 9
        if kind == 1:
            mids = np.concatenate([(mx.GRID4[1:] + mx.GRID4[:-1]) / 2, mx.GRID4, [7, 7.99]])
            b[i] = r.choice(mids, 32) * r.choice([-1, 1], 32) * 2.0 ** int(r.integers(-20, 20))
        elif kind == 2:
            mids = np.concatenate([(mx.GRID8[1:] + mx.GRID8[:-1]) / 2, [448, 449, 460, 511]]).astype(np.float32)
            m = r.choice(mids, 32)
            b[i] = np.where(r.random(32) < 0.5, m, np.nextafter(m, np.float32(r.choice([0, 1e9]))))
        elif kind == 3:
            b[i] = np.nextafter(np.float32(2.0 ** int(r.integers(-10, 10))), np.float32(r.choice([0, 1e9]))) * r.choice([1, -1, 0.25], 32)
        elif kind == 4:
            b[i] = 0
            b[i, 3] = -0.0
        elif kind == 5:
            b[i] *= np.float32(2.0 ** -120) * np.float32(2.0 ** -int(r.integers(0, 28)))
        elif kind == 6:
            b[i] = np.clip(b[i], -1, 1) * np.float32(3.4e38)
        elif kind == 7 and i % 2:
            b[i, int(r.integers(32))] = r.choice([np.inf, -np.inf, np.nan])
    return x


@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (5, 896), (257, 4896), (1, 18944)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_weights_round_to_mxfp4(lib, rows, k, t):
    r = rng(1, rows, k)
    with np.errstate(over="ignore"):
        src = half_types(hard_values(r, rows, k), t)
    codes, scales = guarded(lib, rows * k // 2), guarded(lib, rows * k // 32)
    lib.quantize_mxfp4(lib.to_device(src), {"f32": 0, "f16": 1, "bf16": 2}[t], codes, scales, rows, k)
    want_c, want_s = mx.quantize(widened(src, t), True)
    assert np.array_equal(taken(scales, rows * k // 32, np.uint8, (rows, k // 32)), want_s)
    assert np.array_equal(taken(codes, rows * k // 2, np.uint8, (rows, k // 2)), mx.pack(want_c))


@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (5, 896), (257, 4896), (1, 18944)])
def test_rows_round_to_mxfp8(lib, rows, k):
    x = hard_values(rng(2, rows, k), rows, k)
    codes, scales = guarded(lib, rows * k), guarded(lib, rows * k // 32)
    lib.quantize_mxfp8(lib.to_device(x), codes, scales, rows, k)
    want_c, want_s = mx.quantize(x, False)
    assert np.array_equal(taken(scales, rows * k // 32, np.uint8, (rows, k // 32)), want_s)
    assert np.array_equal(taken(codes, rows * k, np.uint8, (rows, k)), want_c)


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("bf16", [False, True])
def test_values_of_every_code_under_every_scale(lib, four, bf16):
    """bf16: a scale of 3 and more, below which e4m3's subnormals are rounded. Beyond f32's range: infinity."""
    scales = np.arange(3, 256, dtype=np.uint8).repeat(16 if not four else 1).reshape(-1, 1)
    n = len(scales)
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(8, 32), (n // 8 + 1, 1))[:n] if not four else np.tile(np.arange(32, dtype=np.uint8) & 15, (n, 1))
    want = mx.values(codes, scales, four)
    out = guarded(lib, n * 32 * (2 if bf16 else 4))
    dc, ds = lib.to_device(mx.pack(codes) if four else codes), lib.to_device(scales)
    (lib.dequantize_mxfp4 if four else lib.dequantize_mxfp8)(dc, ds, out, lib.T_BF16 if bf16 else lib.T_F32, n, 32)
    got = taken(out, n * 32 * (2 if bf16 else 4), np.uint16 if bf16 else np.float32, (n, 32))
    got = widened(got, "bf16") if bf16 else got
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("rows,n,S", [(1, 32, 0), (1, 896, 1), (3, 896, 0), (301, 3584, 3), (2, 4896, 64), (70, 96, 2), (1, 18944, 1), (2, 32768, 0)])
@pytest.mark.parametrize("out", ["apart", "in place", "none"])
def test_norm_to_mxfp8(lib, rows, n, S, out):
    r = rng(3, rows, n)
    x, w = activations(r, rows, n), (1 + 0.1 * r.standard_normal(n)).astype(np.float32)
    parts = r.standard_normal((S, rows, n)).astype(np.float32)
    want_x, h = mx.norm(x, parts, w, EPS)
    want_c, want_s = mx.quantize(h, False)
    dx = lib.to_device(x)
    xout = {"apart": lib.empty((rows, n)), "in place": dx, "none": None}[out]
    codes, scales = guarded(lib, rows * n), guarded(lib, rows * n // 32)
    lib.rmsnorm_res_mxfp8(dx, lib.to_device(parts) if S else None, S, lib.to_device(w), xout, codes, scales, n, EPS, rows)
    if xout is not None:
        assert np.array_equal(xout.numpy().reshape(rows, n), want_x)
    assert np.array_equal(taken(scales, rows * n // 32, np.uint8, (rows, n // 32)), want_s)
    assert np.array_equal(taken(codes, rows * n, np.uint8, (rows, n)), want_c)


def test_norm_of_rows_that_are_zero_infinite_or_not_a_number(lib):
    r = rng(4)
    x = r.standard_normal((5, 896)).astype(np.float32)
    x[1], x[2, 7], x[3, 890] = 0, np.inf, np.nan
    w = np.ones(896, np.float32)
    codes, scales = lib.empty_bytes(5 * 896), lib.empty_bytes(5 * 28)
    lib.rmsnorm_res_mxfp8(lib.to_device(x), None, 0, lib.to_device(w), None, codes, scales, 896, EPS, 5)
    with np.errstate(invalid="ignore"):
        want_c, want_s = mx.quantize(mx.norm(x, [], w, EPS)[1], False)
    assert np.array_equal(scales.numpy().reshape(5, 28), want_s)
    assert np.array_equal(codes.numpy().reshape(5, 896), want_c)


# Few and many rows, one block of K, K that is no multiple of 128 or 512, features that are no multiple of anything
SHAPES = [(1, 1, 32), (1, 17, 64), (2, 33, 96), (3, 5, 928), (5, 130, 1152), (7, 4608, 896), (15, 96, 4896), (16, 64, 512), (17, 65, 544),
          (31, 257, 160), (33, 100, 4864), (64, 896, 896), (65, 129, 288), (77, 896, 4864), (100, 1, 992), (129, 384, 2080), (200, 1000, 416),
          (257, 515, 896), (301, 600, 1120), (513, 300, 640), (130, 3584, 1184), (1, 3584, 18944), (40, 640, 18944)]


def product_bound(a, w, K):
    return (128 + K / 128 + 64) * 2.0 ** -24 * (np.abs(a) @ np.abs(w).T)


def upload_rows(lib, codes, scales, four=False):
    return lib.to_device(mx.pack(codes) if four else codes), lib.to_device(scales)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(lib, M, N, K):
    r = rng(5, M, N, K)
    (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, N, K)
    a, w = mx.values(ac, asc, False), mx.values(wc, wsc, True)
    out = guarded(lib, M * N * 4)
    before = lib.census()["gemm_mxfp4"]
    lib.gemm_mxfp4_nt(*upload_rows(lib, ac, asc), *upload_rows(lib, wc, wsc, True), out, M, N, K)
    assert lib.census()["gemm_mxfp4"] == before + 1
    got = taken(out, M * N * 4, np.float32, (M, N))
    assert (np.abs(got - a @ w.T) <= product_bound(a, w, K)).all()


@pytest.mark.parametrize("M,N,K", [(1, 17, 64), (7, 896, 4864), (64, 100, 2080), (130, 640, 4896), (257, 515, 896)])
@pytest.mark.parametrize("room", [1, 3, 16])
def test_product_as_parts(lib, M, N, K, room):
    r = rng(6, M, N, K)
    (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, N, K)
    a, w = mx.values(ac, asc, False), mx.values(wc, wsc, True)
    parts = guarded(lib, room * M * N * 4)
    parts.nbytes -= 256
    n = lib.gemm_mxfp4_nt_parts(*upload_rows(lib, ac, asc), *upload_rows(lib, wc, wsc, True), parts, M, N, K)
    parts.nbytes += 256
    assert 1 <= n <= room
    got = taken(parts, room * M * N * 4, np.float32, (room, M, N))
    assert (got[n:].view(np.uint32) == 0xa5a5a5a5).all(), "more parts than were told"
    total = got[:n].astype(np.float64).sum(0)
    assert (np.abs(total - a @ w.T) <= product_bound(a, w, K)).all()


def check_gated(got_c, got_s, a, w, K):
    """Elements next to a border may fall on its other side, and blocks whose largest is next to a power of two may have the other
    scale: by as much as the product's bound (a gate's slope is below 1.1, so it and the up value each pass on theirs)."""
    gu = a @ w.T
    bound = product_bound(a, w, K)
    ff = gu.shape[1] // 2
    act = mx.swiglu(gu)
    # |d act| <= 1.1 |up| d gate + |silu(gate)| d up, and eight roundings of the gate's own arithmetic
    off = 1.1 * np.abs(gu[:, ff:]) * bound[:, :ff] + np.abs(act / np.where(gu[:, ff:] == 0, 1, gu[:, ff:])) * bound[:, ff:] + np.abs(act) * 2.0 ** -20 + 1e-37
    v = mx.values(got_c, got_s, False)
    # a value in [448, 512) times the scale became 448; one rounding of the element: half a step, of the value or of the lowest exponent's
    step = np.maximum(np.abs(act) * 2.0 ** -4, (2.0 ** (got_s.astype(np.float64) - 127) * 2.0 ** -10).repeat(32, 1))
    top = (2.0 ** (got_s.astype(np.float64) - 127) * 448).repeat(32, 1)
    err = np.abs(v - act) - np.where(np.abs(act) > top, np.abs(act) - top, 0)
    assert (err <= step + off).all()
    # the scale itself: of the largest magnitude, which is known to within `off`
    big = np.abs(act).reshape(len(act), -1, 32).max(-1)
    o = off.reshape(len(act), -1, 32).max(-1)
    lo, hi = (np.maximum(np.floor(np.log2(np.maximum(b, 2.0 ** -140))) + 119, 0) for b in (big - o, big + o))
    assert ((lo <= got_s) & (got_s <= hi)).all()
    # and nearly all are what 64 bits give
    want_c, want_s = mx.quantize(act.astype(np.float32), False)
    assert (want_s != got_s).mean() < 0.01 and (want_c != got_c)[(want_s == got_s).repeat(32, 1)].mean() < 0.01


@pytest.mark.parametrize("M,ff,K", [(1, 32, 32), (1, 4864, 896), (3, 96, 544), (16, 64, 512), (17, 160, 928), (40, 416, 4896), (77, 1216, 896),
                                    (130, 352, 1152), (257, 608, 416), (301, 4864, 896), (513, 96, 640)])
def test_gated_product_to_mxfp8(lib, M, ff, K):
    r = rng(7, M, ff, K)
    (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, 2 * ff, K)
    wsc = (wsc + 3).astype(np.uint8)          # (gates of order one: both of the sigmoid's sides)
    codes, scales = guarded(lib, M * ff), guarded(lib, M * ff // 32)
    lib.gemm_mxfp4_nt_swiglu(*upload_rows(lib, ac, asc), *upload_rows(lib, wc, wsc, True), codes, scales, M, ff, K)
    check_gated(taken(codes, M * ff, np.uint8, (M, ff)), taken(scales, M * ff // 32, np.uint8, (M, ff // 32)),
                mx.values(ac, asc, False), mx.values(wc, wsc, True), K)


TOKENS = [(1, 32), (3, 64), (17, 96), (16, 512), (896, 896), (1000, 544), (33, 4896), (896, 4864), (4608, 3584), (257, 18944), (20000, 160),
          (33280, 160), (16640, 3584), (16656, 1184), (16650, 1184), (40, 65536)]


# few tiles over a long K: parts that are added up, and gated, by a launch of their own; rows of no whole number of 16 bytes
@pytest.mark.parametrize("M,N,K", [(17, 1, 9408), (23, 3, 18496), (103, 1113, 2560), (200, 6, 3328), (130, 141, 4896), (33, 5, 65536)])
def test_product_of_few_tiles(lib, M, N, K):
    r = rng(71, M, N, K)
    ac, asc = rows8(r, M, K)
    wc, wsc = weight(r, N, K)
    bufs = upload_rows(lib, ac, asc) + upload_rows(lib, wc, wsc, True)
    out = guarded(lib, M * N * 4)
    lib.gemm_mxfp4_nt(*bufs, out, M, N, K)
    a, w = mx.values(ac, asc, False), mx.values(wc, wsc, True)
    assert np.all(np.abs(taken(out, M * N * 4, np.float32, (M, N)) - a @ w.T) <= product_bound(a, w, K))
    room = 16
    parts = guarded(lib, room * M * N * 4)
    parts.nbytes, nbytes = room * M * N * 4, parts.nbytes
    n = lib.gemm_mxfp4_nt_parts(*bufs, parts, M, N, K)
    parts.nbytes = nbytes
    got = taken(parts, room * M * N * 4, np.float32, (room, M, N))[:n].astype(np.float64).sum(0)
    assert n >= 1 and np.all(np.abs(got - a @ w.T) <= product_bound(a, w, K))
    for b in bufs + (out, parts):
        b.free()


@pytest.mark.parametrize("M,ff,K", [(1, 32, 1536), (12, 32, 10368), (16, 96, 4096), (7, 4128, 2048), (19, 32, 9408), (282, 32, 11552), (130, 160, 2720), (40, 864, 3584), (5, 32, 65536)])
def test_gated_product_of_few_tiles(lib, M, ff, K):
    r = rng(73, M, ff, K)
    ac, asc = rows8(r, M, K)
    wc, wsc = weight(r, 2 * ff, K)
    bufs = upload_rows(lib, ac, asc) + upload_rows(lib, wc, wsc, True)
    oc, os_ = guarded(lib, M * ff), guarded(lib, M * ff // 32)
    lib.gemm_mxfp4_nt_swiglu(*bufs, oc, os_, M, ff, K)
    check_gated(taken(oc, M * ff, np.uint8, (M, ff)), taken(os_, M * ff // 32, np.uint8, (M, ff // 32)), mx.values(ac, asc, False), mx.values(wc, wsc, True), K)
    for b in bufs + (oc, os_):
        b.free()


@pytest.mark.parametrize("g", [0.0, 1e-30, -1e-3, 5.0, -20.0, 60.0, -60.0, -86.0, 3e4, 3e38])
def test_gate_of_small_and_large_numbers(lib, g):
    """One row and K = 32: gate values g times 1, 2, 4 (by the weights' elements), up values of order one. Eight roundings of the gate's arithmetic."""
    K, ff = 32, 32
    a = np.zeros((1, K), np.float32)
    a[0, 0], a[0, 1] = g, 1.0
    ac, asc = mx.quantize(a, False)
    w = np.zeros((2 * ff, K), np.float32)
    w[:ff, 0] = np.resize([1, 2, 4, 1, 1], ff)
    w[ff:, 1] = np.resize([1, 1.5, -3], ff)
    if abs(g) > 1e3 or abs(g) < 1e-3:      # (the block has one scale: the gate's number alone)
        w[ff:, 1], w[ff:, 0] = 0, 0.5
    wc, wsc = mx.quantize(w, True)
    bufs = upload_rows(lib, ac, asc) + upload_rows(lib, wc, wsc, True)
    oc, os_ = guarded(lib, ff), guarded(lib, 1)
    lib.gemm_mxfp4_nt_swiglu(*bufs, oc, os_, 1, ff, K)
    gu = mx.values(ac, asc, False) @ mx.values(wc, wsc, True).T
    with np.errstate(over="ignore", invalid="ignore"):
        act = mx.swiglu(gu)
    c, s = taken(oc, ff, np.uint8, (1, ff)), taken(os_, 1, np.uint8, (1, 1))
    if np.abs(act).max() > 3.4e38:
        assert s[0, 0] == 255 and not c.any()
    else:
        v = mx.values(c, s, False)
        step = np.maximum(np.abs(act) * 2.0 ** -4, 2.0 ** (float(s[0, 0]) - 127 - 10))
        top = 2.0 ** (float(s[0, 0]) - 127) * 448
        assert np.all(np.abs(v - act) - np.maximum(np.abs(act) - top, 0) <= step + np.abs(act) * 2.0 ** -20 + 1e-37)
    for b in bufs + (oc, os_):
        b.free()


@pytest.mark.parametrize("N,K", TOKENS)
def test_token_product(lib, N, K):
    r = rng(8, N, K)
    x, (wc, wsc) = activations(r, 1, K), weight(r, N, K)
    w = mx.values(wc, wsc, True)
    out = guarded(lib, 4 * N)
    lib.gemv_mxfp4(lib.to_device(x), *upload_rows(lib, wc, wsc, True), out, N, K)
    got = taken(out, 4 * N, np.float32, (N,))
    big = np.abs(x[0].astype(np.float64)).reshape(-1, 32).max(-1).repeat(32)
    bound = product_bound(x.astype(np.float64), w, K)[0] + 2.0 ** -38 * (np.abs(w) @ big)
    assert (np.abs(got - w @ x[0].astype(np.float64)) <= bound).all()


@pytest.mark.parametrize("N,K", [(1, 32), (17, 96), (896, 896), (1152, 896), (130, 4896), (4608, 3584), (33280, 160), (16640, 2080), (48, 18944), (40, 65536)])
@pytest.mark.parametrize("delta", [False, True])
def test_token_product_behind_a_norm(lib, N, K, delta):
    """Row totals are multiplied by 1 / rms, whose own error is K / 64 additions a lane and 14 more (2^-24 each, half of it in the root),
    and the numbers by the norm's weights: two roundings each."""
    r = rng(20, N, K)
    x, d, nw, (wc, wsc) = activations(r, 1, K)[0], activations(r, 1, K)[0], (1 + 0.1 * r.standard_normal(K)).astype(np.float32), weight(r, N, K)
    w, s = mx.values(wc, wsc, True), x + d if delta else x
    s64 = s.astype(np.float64)
    h = s64 / np.sqrt((s64 * s64).mean() + EPS) * nw
    out, xout = guarded(lib, 4 * N), guarded(lib, 4 * K)
    lib.gemv_mxfp4_rmsnorm(lib.to_device(x), lib.to_device(d) if delta else None, lib.to_device(nw), xout, *upload_rows(lib, wc, wsc, True), out, N, K, EPS)
    assert np.array_equal(taken(xout, 4 * K, np.float32, (K,)), s)
    got = taken(out, 4 * N, np.float32, (N,))
    rel = (K / 64 + 20) * 2.0 ** -24
    assert (np.abs(got - w @ h) <= product_bound(h[None], w, K)[0] + rel * (np.abs(w) @ np.abs(h))).all()


@pytest.mark.parametrize("ff,K", [(1, 32), (17, 96), (896, 896), (4864, 896), (130, 4896), (2432, 3584), (33280, 160), (16640, 2080), (48, 18944), (20, 65536)])
@pytest.mark.parametrize("delta", [False, True])
def test_gated_token_product_behind_a_norm(lib, ff, K, delta):
    r = rng(21, ff, K)
    x, d, nw, (wc, wsc) = activations(r, 1, K)[0], activations(r, 1, K)[0], (1 + 0.1 * r.standard_normal(K)).astype(np.float32), weight(r, 2 * ff, K)
    w, s = mx.values(wc, wsc, True), (x + d if delta else x).astype(np.float64)
    h = s / np.sqrt((s * s).mean() + EPS) * nw
    out = guarded(lib, 4 * ff)
    lib.gemv_mxfp4_rmsnorm_gateup(lib.to_device(x), lib.to_device(d) if delta else None, lib.to_device(nw), None, *upload_rows(lib, wc, wsc, True), out,
                                  2 * ff, K, EPS)
    got = taken(out, 4 * ff, np.float32, (ff,))
    gu = w @ h
    off = product_bound(h[None], w, K)[0] + (K / 64 + 20) * 2.0 ** -24 * (np.abs(w) @ np.abs(h))
    g, u = gu[:ff], gu[ff:]
    silu = g / (1 + np.exp(-g))
    # a gate's slope is below 1.1; eight roundings of the gate's own arithmetic
    assert (np.abs(got - silu * u) <= 1.1 * np.abs(u) * off[:ff] + np.abs(silu) * off[ff:] + 1.2 * off[:ff] * off[ff:] + np.abs(silu * u) * 2.0 ** -20 + 1e-37).all()


@pytest.mark.parametrize("D,heads,S", [(64, 14, 16), (64, 14, 5), (128, 28, 8), (128, 2, 3), (64, 4, 1), (64, 2, 9), (128, 64, 7)])
@pytest.mark.parametrize("N", [1, 130, 4640])
def test_token_product_of_the_attentions_splits(lib, orc, D, heads, S, N):
    """Made-up partials, some of splits without a key: the row that the bf16 product merges (through the identity, exactly) and 64 bits. A split's weight e^(m - M), |m - M| up to 60, has 60 / ln 2 + 4 roundings (of the
    argument, and of the exponential), in the sums above and below; each sum has one more for each split, the quotient one."""
    r, K = rng(D, heads, S, N), heads * D
    m = r.uniform(-30, 30, (heads, S)).astype(np.float32)
    l = r.uniform(0.5, 64, (heads, S)).astype(np.float32)
    acc = (r.standard_normal((heads, S, D)) * l[:, :, None]).astype(np.float32)
    if S > 2:
        for h, s in enumerate(r.integers(1, S, heads)):
            m[h, s], l[h, s], acc[h, s] = -np.inf, 0, 0
    part = lib.to_device(np.concatenate([m.ravel(), l.ravel(), acc.ravel()]))
    codes, scales = weight(r, N, K)
    wc, ws = upload_rows(lib, codes, scales, True)
    x, y, eye = lib.empty(K), lib.empty(N), lib.to_device(orc.to_bf16(np.eye(K, dtype=np.float32)))
    lib.gemv_bf16_row_attn(part, S, heads, D, eye, x, K, K)
    lib.gemv_mxfp4_attn(part, S, heads, D, wc, ws, y, N, K)
    merged, W = x.numpy().astype(np.float64), mx.values(codes, scales, True)
    assert np.all(np.abs(y.numpy() - W @ merged) <= product_bound(merged[None], W, K)[0])
    w64 = np.exp(m.astype(np.float64) - m.max(axis=1, keepdims=True))
    row = ((w64[:, :, None] * acc).sum(axis=1) / (w64 * l).sum(axis=1)[:, None]).reshape(K)
    size = ((w64[:, :, None] * np.abs(acc)).sum(axis=1) / (w64 * l).sum(axis=1)[:, None]).reshape(K)
    bound = (128 + K / 128 + 64 + 2 * (60 / np.log(2) + 4 + S) + 1) * 2.0 ** -24 * (np.abs(W) @ size)
    assert np.all(np.abs(y.numpy() - W @ row) <= bound)
    for S_, h_ in ((17 if D == 64 else 9, heads), (0, heads), (S, heads + 1)):
        with pytest.raises(Exception):
            lib.gemv_mxfp4_attn(part, S_, h_, D, wc, ws, y, N, K)
    for b in (part, wc, ws, x, y, eye):
        b.free()


def test_token_product_is_that_of_the_rows_apart(lib):
    """A row of the weight gives the same sum whatever rows lie beside it (blocks of one launch shape)."""
    r = rng(22)
    x, (wc, wsc) = lib.to_device(activations(r, 1, 896)), weight(r, 96, 896)
    whole, part = lib.empty(96), lib.empty(32)
    lib.gemv_mxfp4(x, *upload_rows(lib, wc, wsc, True), whole, 96, 896)
    lib.gemv_mxfp4(x, *upload_rows(lib, wc[32:64], wsc[32:64], True), part, 32, 896)
    assert np.array_equal(whole.numpy()[32:64], part.numpy())


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("M,K", [(1, 896), (5, 896), (70, 896), (70, 1184)])
def test_scales_anywhere(lib, M, K, off):
    """Scale bytes at odd addresses, of both operands: products and the decode product."""
    r, N = rng(23, M, K), 130
    (ac, asc), (wc, wsc), x = rows8(r, M, K), weight(r, N, K), activations(r, 1, K)
    a, w = mx.values(ac, asc, False), mx.values(wc, wsc, True)

    def shifted(scales):
        b = lib.to_device(np.concatenate([np.full(off, 255, np.uint8), scales.reshape(-1)]))
        b.ptr += off
        return b
    da, dw, sa, sw, out = lib.to_device(ac), lib.to_device(mx.pack(wc)), shifted(asc), shifted(wsc), lib.empty((M, N))
    lib.gemm_mxfp4_nt(da, sa, dw, sw, out, M, N, K)
    assert (np.abs(out.numpy() - a @ w.T) <= product_bound(a, w, K)).all()
    y = lib.empty(N)
    lib.gemv_mxfp4(lib.to_device(x), dw, sw, y, N, K)
    big = np.abs(x[0].astype(np.float64)).reshape(-1, 32).max(-1).repeat(32)
    assert (np.abs(y.numpy() - w @ x[0]) <= product_bound(x.astype(np.float64), w, K)[0] + 2.0 ** -38 * (np.abs(w) @ big)).all()
    for b in (sa, sw):
        b.ptr -= off


@pytest.mark.parametrize("kind", ["spread", "largest", "smallest", "one outlier"])
def test_token_product_of_hard_rows(lib, kind):
    """f32 sums of the row's numbers as they are: magnitudes all over a block, at both ends of f32, and one that dwarfs its
    neighbours under weights of zero."""
    r, N, K = rng(24), 64, 1152
    x, (wc, wsc) = r.standard_normal((1, K)).astype(np.float32), weight(r, N, K)
    if kind == "spread":
        x *= 2.0 ** r.integers(-22, 1, (1, K)).astype(np.float32)
    elif kind == "largest":
        x *= np.float32(2.0 ** 125) / np.abs(x).max()
        wsc = (wsc - 8).astype(np.uint8)
    elif kind == "smallest":
        x *= np.float32(2.0 ** -100)
        wsc = (wsc + 20).astype(np.uint8)
    else:
        x[0, 5::32] = 2.0 ** 20
        wc[:, 5::32] &= 8
    w, x64 = mx.values(wc, wsc, True), x.astype(np.float64)
    out = lib.empty(N)
    lib.gemv_mxfp4(lib.to_device(x), *upload_rows(lib, wc, wsc, True), out, N, K)
    big = np.abs(x64[0]).reshape(-1, 32).max(-1).repeat(32)
    bound = product_bound(x64, w, K)[0] + np.abs(w) @ np.maximum(2.0 ** -48 * big, 2.0 ** -128)
    assert (np.abs(out.numpy() - w @ x64[0]) <= bound).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_token_product_of_a_row_that_is_not_finite(lib, bad):
    r = rng(25)
    x, (wc, wsc) = activations(r, 1, 896), weight(r, 100, 896)
    x[0, 777] = bad
    out = lib.empty(100)
    lib.gemv_mxfp4(lib.to_device(x), *upload_rows(lib, wc, wsc, True), out, 100, 896)
    assert np.isnan(out.numpy()).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_token_product_of_small_and_large_numbers(lib, scale):
    r = rng(9)
    x, (wc, wsc) = activations(r, 1, 896) * np.float32(scale), weight(r, 100, 896)
    w = mx.values(wc, wsc, True)
    out = lib.empty(100)
    lib.gemv_mxfp4(lib.to_device(x), *upload_rows(lib, wc, wsc, True), out, 100, 896)
    big = np.abs(x[0].astype(np.float64)).reshape(-1, 32).max(-1).repeat(32)
    bound = product_bound(x.astype(np.float64), w, 896)[0] + 2.0 ** -38 * (np.abs(w) @ big)
    assert (np.abs(out.numpy() - w @ x[0].astype(np.float64)) <= bound).all()


@pytest.mark.parametrize("M,N,K", [(5, 70, 416), (200, 300, 928)])
def test_not_a_number_stays_with_its_row(lib, M, N, K):
    """A block with scale 255, or an element that is NaN, makes its own row of the result NaN and no other; blocks at the ends of the
    rows are what the tiles' edges read."""
    r = rng(10, M, N)
    (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, N, K)
    clean = mx.values(ac, asc, False) @ mx.values(wc, wsc, True).T
    asc[M - 1, -1], wsc[2, 0], ac[1, K - 1] = 255, 255, 0x7f
    wsc[N - 1, -1] = 255
    out = lib.empty((M, N))
    lib.gemm_mxfp4_nt(*upload_rows(lib, ac, asc), *upload_rows(lib, wc, wsc, True), out, M, N, K)
    got = out.numpy()
    nan = np.zeros((M, N), bool)
    nan[[1, M - 1]] = True
    nan[:, [2, N - 1]] = True
    assert np.array_equal(np.isnan(got), nan)
    assert np.allclose(got[~nan], clean[~nan], rtol=1e-4, atol=1e-4 * np.abs(clean).max())
    y = lib.empty(N)
    lib.gemv_mxfp4(lib.to_device(activations(r, 1, K)), *upload_rows(lib, wc, wsc, True), y, N, K)
    assert np.array_equal(np.isnan(y.numpy()), nan[0])


@pytest.mark.parametrize("M", [1, 9, 77])
def test_layer_of_a_prompt(lib, M):
    """The calls of a feed-forward layer one after the other: norm, gated product, down projection in parts, norm of the next
    layer; each held to 64 bits on what the call before it wrote."""
    r = rng(11, M)
    E, F = 896, 1216
    x, w1, w2 = activations(r, M, E), (1 + 0.1 * r.standard_normal(E)).astype(np.float32), (1 + 0.1 * r.standard_normal(E)).astype(np.float32)
    (gc, gs), (dc, ds) = weight(r, 2 * F, E), weight(r, E, F)
    hc, hs, fc, fs = (lib.empty_bytes(n) for n in (M * E, M * E // 32, M * F, M * F // 32))
    dx, parts = lib.to_device(x), lib.empty((8, M, E))
    lib.rmsnorm_res_mxfp8(dx, None, 0, lib.to_device(w1), None, hc, hs, E, EPS, M)
    lib.gemm_mxfp4_nt_swiglu(hc, hs, *upload_rows(lib, gc, gs, True), fc, fs, M, F, E)
    n = lib.gemm_mxfp4_nt_parts(fc, fs, *upload_rows(lib, dc, ds, True), parts, M, E, F)
    first = hc.numpy().reshape(M, E), hs.numpy().reshape(M, -1)
    lib.rmsnorm_res_mxfp8(dx, parts, n, lib.to_device(w2), dx, hc, hs, E, EPS, M)
    want = mx.quantize(mx.norm(x, [], w1, EPS)[1], False)
    assert np.array_equal(first[0], want[0]) and np.array_equal(first[1], want[1])
    f = fc.numpy().reshape(M, F), fs.numpy().reshape(M, -1)
    check_gated(*f, mx.values(*first, False), mx.values(gc, gs, True), E)
    p = parts.numpy()[:n]
    a, w = mx.values(*f, False), mx.values(dc, ds, True)
    assert (np.abs(p.astype(np.float64).sum(0) - a @ w.T) <= product_bound(a, w, F)).all()
    want_x, h = mx.norm(x, p, w2, EPS)
    want = mx.quantize(h, False)
    assert np.array_equal(dx.numpy().reshape(M, E), want_x)
    assert np.array_equal(hc.numpy().reshape(M, E), want[0]) and np.array_equal(hs.numpy().reshape(M, -1), want[1])


@pytest.mark.parametrize("N,K", [(131136, 65536), ((1 << 21) + 64, 4096)])
def test_weights_beyond_four_gigabytes(lib, N, K):
    """Rows of ones, the last 40 of them random: every kernel's offsets into a weight of more than 2^32 bytes."""
    r, tail = rng(81, N), 40
    codes, scales = weight(r, tail, K)
    wc, ws = lib.empty_bytes(N * K // 2), lib.empty_bytes(N * K // 32)
    lib._chk(lib.c.tlhip_fill_u32(wc.ptr, 0x22222222, N * K // 8))
    lib._chk(lib.c.tlhip_fill_u32(ws.ptr, 0x7f7f7f7f, N * K // 128))
    packed = np.ascontiguousarray(mx.pack(codes))
    lib._chk(lib.c.tlhip_memcpy_h2d(wc.ptr + (N - tail) * K // 2, packed.ctypes.data, packed.nbytes))
    scales = np.ascontiguousarray(scales)
    lib._chk(lib.c.tlhip_memcpy_h2d(ws.ptr + (N - tail) * K // 32, scales.ctypes.data, scales.nbytes))
    w = np.concatenate([np.ones((1, K)), mx.values(codes, scales, True)])
    a = activations(r, 17, K)
    x, y = lib.to_device(a[0]), lib.empty(N)
    lib.gemv_mxfp4(x, wc, ws, y, N, K)
    want, bound = (a[:1].astype(np.float64) @ w.T)[0], product_bound(a[:1].astype(np.float64), w, K)[0]
    got = y.numpy()
    assert np.all(np.abs(got[:N - tail] - want[0]) <= bound[0]) and np.all(np.abs(got[N - tail:] - want[1:]) <= bound[1:])
    ac, asc = mx.quantize(a, False)
    av = mx.values(ac, asc, False)
    want, bound = av @ w.T, product_bound(av, w, K)
    da, out = upload_rows(lib, ac, asc), lib.empty((17, N))
    for M in (3, 17):
        lib.gemm_mxfp4_nt(*da, wc, ws, out, M, N, K)
        got = out.numpy().reshape(17, N)[:M]
        assert np.all(np.abs(got[:, :N - tail] - want[:M, :1]) <= bound[:M, :1])
        assert np.all(np.abs(got[:, N - tail:] - want[:M, 1:]) <= bound[:M, 1:])
    ff = N // 2                                  # gate rows of ones, up rows of ones and the random ones
    oc, os_ = lib.empty_bytes(17 * ff), lib.empty_bytes(17 * ff // 32)
    up = 2.0 ** -14                              # (sums of thousands of numbers of order one: a row small enough for the gate)
    ac, asc = mx.quantize(a * np.float32(up), False)
    av = mx.values(ac, asc, False)
    for b in da:
        b.free()
    da = upload_rows(lib, ac, asc)
    gu = av @ w.T
    bound = product_bound(av, w, K)
    for M in (3, 17):
        lib.gemm_mxfp4_nt_swiglu(*da, wc, ws, oc, os_, M, ff, K)
        v = mx.values(oc.numpy(np.uint8)[:M * ff].reshape(M, ff)[:, ff - 64:], os_.numpy(np.uint8)[:M * ff // 32].reshape(M, ff // 32)[:, -2:], False)
        g, u = gu[:M, :1], np.concatenate([np.repeat(gu[:M, :1], 64 - tail, 1), gu[:M, 1:]], 1)
        act = mx.swiglu(np.concatenate([np.repeat(g, 64, 1), u], 1))
        bu = np.concatenate([np.repeat(bound[:M, :1], 64 - tail, 1), bound[:M, 1:]], 1)
        off = 1.1 * np.abs(u) * bound[:M, :1] + np.abs(act / np.where(u == 0, 1, u)) * bu + np.abs(act) * 2.0 ** -20 + 1e-37
        top = np.abs(act).reshape(M, 2, 32).max(-1).repeat(32, 1)
        # one rounding of an element: half a step of its own, or 2^-10 of the scale, which is at most 2^-8 of the largest;
        # what lies in [448, 512) times the scale became 448, at most an eighth off
        step = np.maximum(np.abs(act) * 2.0 ** -4, top * 2.0 ** -18)
        step = np.where(np.abs(act) > top * 0.875 - off, np.abs(act) * 0.125, step)
        assert np.all(np.abs(v - act) <= step + off)
    for b in da + (wc, ws, x, y, out, oc, os_):
        b.free()


@pytest.mark.parametrize("M,N,K", [(1, 896, 4864), (7, 896, 4864), (33, 416, 2080), (130, 896, 4864)])
def test_recorded_product(fresh_lib, recorded, M, N, K):
    """Recorded ahead of any eager call, replayed with other work between: what the eager call gives, or its parts in another
    order."""
    lib, r = fresh_lib, rng(12, M)
    (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, N, K)
    a, w = mx.values(ac, asc, False), mx.values(wc, wsc, True)
    da, dw, out = upload_rows(lib, ac, asc), upload_rows(lib, wc, wsc, True), lib.empty((M, N))
    for got in recorded(lambda: lib.gemm_mxfp4_nt(*da, *dw, out, M, N, K), out):
        assert (np.abs(got.reshape(M, N) - a @ w.T) <= product_bound(a, w, K)).all()


def test_recorded_layer(fresh_lib, recorded):
    lib, r = fresh_lib, rng(13)
    M, E, F = 33, 896, 608
    x, nw = lib.to_device(activations(r, M, E)), lib.to_device(np.ones(E, np.float32))
    g, d = upload_rows(lib, *weight(r, 2 * F, E), True), upload_rows(lib, *weight(r, E, F), True)
    hc, hs, fc, fs = (lib.empty_bytes(n) for n in (M * E, M * E // 32, M * F, M * F // 32))
    y, tok, row = lib.empty((M, E)), lib.empty(E), lib.to_device(activations(r, 1, F))
    both = lib.empty(M * E + E)

    def layer():
        lib.rmsnorm_res_mxfp8(x, None, 0, nw, None, hc, hs, E, EPS, M)
        lib.gemm_mxfp4_nt_swiglu(hc, hs, *g, fc, fs, M, F, E)
        lib.gemm_mxfp4_nt(fc, fs, *d, y, M, E, F)
        lib.gemv_mxfp4(row, *d, tok, E, F)
        lib._chk(lib.c.tlhip_memcpy_d2d_async(both.ptr, y.ptr, y.nbytes))
        lib._chk(lib.c.tlhip_memcpy_d2d_async(both.ptr + y.nbytes, tok.ptr, tok.nbytes))

    replays = recorded(layer, both)
    layer()
    lib.sync()
    eager = both.numpy()
    scale = np.abs(eager).max()
    for got in replays:
        assert np.abs(got - eager).max() <= 1e-5 * scale
    assert np.array_equal(replays[0], replays[1]) and np.array_equal(replays[0], replays[2])


@pytest.mark.parametrize("M,N,K", [(40, 192, 8192), (20, 576, 9408), (9, 192, 8224)])
def test_recorded_products_in_parts(fresh_lib, recorded, M, N, K):
    """Behind an eager call, so that there is a workspace: products of few tiles in parts, plain and gated, replayed with other work on
    the same workspace between: the eager call's bytes."""
    lib, r = fresh_lib, rng(91, M, K)
    da, dw = upload_rows(lib, *rows8(r, M, K)), upload_rows(lib, *weight(r, N, K), True)
    other = upload_rows(lib, *rows8(r, 60, K))
    y, ff = lib.empty((M, N)), N // 2
    codes, scales, dump = lib.empty_bytes(M * ff), lib.empty_bytes(M * ff // 32), lib.empty((60, N))
    both = lib.empty_bytes(M * N * 4 + M * ff + M * ff // 32)

    def calls():
        lib.gemm_mxfp4_nt(*da, *dw, y, M, N, K)
        lib.gemm_mxfp4_nt_swiglu(*da, *dw, codes, scales, M, ff, K)
        lib.gemm_mxfp4_nt(*other, *dw, dump, 60, N, K)
        at = both.ptr
        for b, n in ((y, M * N * 4), (codes, M * ff), (scales, M * ff // 32)):
            lib._chk(lib.c.tlhip_memcpy_d2d_async(at, b.ptr, n))
            at += n

    calls()
    lib.sync()
    eager = both.numpy().copy()
    for got in recorded(calls, both):
        assert np.array_equal(got, eager)


def test_products_are_deterministic(lib):
    r = rng(14)
    for M, N, K in [(1, 4608, 3584), (7, 896, 4864), (129, 896, 4864)]:
        (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, N, K)
        da, dw, out = upload_rows(lib, ac, asc), upload_rows(lib, wc, wsc, True), lib.empty((M, N))
        got = []
        for _ in range(3):
            lib.gemm_mxfp4_nt(*da, *dw, out, M, N, K)
            got.append(out.numpy())
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_results_over_operands_are_refused(lib):
    """Every product, with its result in the place of each thing it reads (or writes beside it)."""
    b = lib.empty_bytes(1 << 16)
    c, n = lib.c, C.c_int(0)
    p = [b.ptr + 4096 * i for i in range(8)]
    products = [                                  # call of (operands, result), how many operands
        (c.tlhip_gemv_mxfp4, lambda o, y: (*o, y, 1, 32), 3),
        (c.tlhip_gemv_mxfp4_attn, lambda o, y: (o[0], 2, 2, 64, o[1], o[2], y, 1, 128), 3),
        (c.tlhip_gemv_mxfp4_rmsnorm, lambda o, y: (*o, y, 1, 32, 1e-6), 6),
        (c.tlhip_gemv_mxfp4_rmsnorm, lambda o, y: (*o[:3], y, *o[3:], 1, 32, 1e-6), 6),              # (the sum's row)
        (c.tlhip_gemv_mxfp4_rmsnorm_gateup, lambda o, y: (*o, y, 2, 32, 1e-6), 6),
        (c.tlhip_gemv_mxfp4_rmsnorm_gateup, lambda o, y: (*o[:3], y, *o[3:], 2, 32, 1e-6), 6),
        (c.tlhip_gemm_mxfp4_nt, lambda o, y: (*o, y, 1, 32, 32), 4),
        (c.tlhip_gemm_mxfp4_nt_parts, lambda o, y: (*o, y, 4096, 1, 32, 32, C.byref(n)), 4),
        (c.tlhip_gemm_mxfp4_nt_swiglu, lambda o, y: (*o[:4], y, o[4], 1, 32, 32), 5),
        (c.tlhip_gemm_mxfp4_nt_swiglu, lambda o, y: (*o, y, 1, 32, 32), 5),
    ]
    before = lib.census()
    for fn, args, operands in products:
        for i in range(operands):
            assert fn(*args(p[:operands], p[i])) == -2, (fn.__name__, i)
            assert lib.last_error().startswith(fn.__name__)
    assert lib.census() == before


def test_refusals(lib):
    b, odd = lib.empty_bytes(1 << 16), C.c_void_p(0)
    p, n = b.ptr, C.c_int(0)
    odd = p + 4
    EINVAL, EUNSUPPORTED = -2, -3
    c = lib.c
    cases = [
        (c.tlhip_quantize_mxfp4, (None, 0, p, p, 1, 32), EINVAL), (c.tlhip_quantize_mxfp4, (p, 3, p, p, 1, 32), EUNSUPPORTED),
        (c.tlhip_quantize_mxfp4, (p, 0, p, p, 0, 32), EINVAL), (c.tlhip_quantize_mxfp4, (p, 0, p, p, 1, 33), EINVAL),
        (c.tlhip_quantize_mxfp4, (p, 0, p, p, 1, 0), EINVAL), (c.tlhip_quantize_mxfp4, (odd, 0, p, p, 1, 32), EINVAL),
        (c.tlhip_quantize_mxfp4, (p, 0, odd, p, 1, 32), EINVAL), (c.tlhip_quantize_mxfp4, (p, 0, p, p, 1 << 62, 1 << 20), EUNSUPPORTED),
        (c.tlhip_quantize_mxfp8, (p, None, p, 1, 32), EINVAL), (c.tlhip_quantize_mxfp8, (p, p, p, 1, 16), EINVAL),
        (c.tlhip_quantize_mxfp8, (p, p, p, -1, 32), EINVAL), (c.tlhip_quantize_mxfp8, (p, odd, p, 1, 32), EINVAL),
        (c.tlhip_dequantize_mxfp4, (p, p, p, 1, 1, 32), EUNSUPPORTED), (c.tlhip_dequantize_mxfp4, (p, None, p, 0, 1, 32), EINVAL),
        (c.tlhip_dequantize_mxfp8, (p, p, odd, 0, 1, 32), EINVAL), (c.tlhip_dequantize_mxfp8, (p, p, p, 0, 1, 40), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 1, p, None, p, p, 32, 1e-6, 1), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, p, 1, p, p, p, p, 32, 1e-6, 1), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, p, None, p, p, 40, 1e-6, 1), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, p, None, p, p, 32800, 1e-6, 1), EUNSUPPORTED),
        (c.tlhip_rmsnorm_res_mxfp8, (p, p, 65, p, None, p, p, 32, 1e-6, 1), EUNSUPPORTED),
        (c.tlhip_rmsnorm_res_mxfp8, (p, p, -1, p, None, p, p, 32, 1e-6, 1), EUNSUPPORTED),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, p, odd, p, p, 32, 1e-6, 1), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, p, None, p, p, 32, 1e-6, (1 << 20) + 1), EUNSUPPORTED),
        (c.tlhip_gemm_mxfp4_nt, (p, p, p, p, p, 1 << 20, 1 << 24, 32), EUNSUPPORTED),
        (c.tlhip_gemm_mxfp4_nt_swiglu, (p, p, p, p, p, p, 1 << 20, 1 << 20, 32), EUNSUPPORTED),
        (c.tlhip_gemv_mxfp4_attn, (p, 1, 1, 32, p, p, p, 1, 32), EINVAL), (c.tlhip_gemv_mxfp4_attn, (p, 17, 2, 64, p, p, p, 1, 128), EUNSUPPORTED),
        (c.tlhip_gemv_mxfp4_attn, (p, 1, 1, 64, p, p, p, 1, 64), EUNSUPPORTED), (c.tlhip_gemv_mxfp4_attn, (None, 1, 2, 64, p, p, p, 1, 128), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, p, None, p, p, 32, 1e-6, 0), EINVAL),
        (c.tlhip_gemv_mxfp4, (p, p, p, None, 1, 32), EINVAL), (c.tlhip_gemv_mxfp4, (p, p, p, p, 1, 48), EINVAL),
        (c.tlhip_gemv_mxfp4, (p, odd, p, p, 1, 32), EINVAL), (c.tlhip_gemv_mxfp4, (p, p, p, p, 0, 32), EINVAL),
        (c.tlhip_gemv_mxfp4, (p, p, p, p, 1 << 40, 32), EUNSUPPORTED), (c.tlhip_gemv_mxfp4, (p, p, p, p, 1, 65568), EUNSUPPORTED),
        (c.tlhip_gemv_mxfp4_rmsnorm, (p, None, None, None, p, p, p, 1, 32, 1e-6), EINVAL),
        (c.tlhip_gemv_mxfp4_rmsnorm, (p, odd, p, None, p, p, p, 1, 32, 1e-6), EINVAL),
        (c.tlhip_gemv_mxfp4_rmsnorm, (p, None, p, p, p, p, p, 1, 32, 1e-6), EINVAL),
        (c.tlhip_gemv_mxfp4_rmsnorm_gateup, (p, None, p, None, p, p, p, 3, 32, 1e-6), EINVAL),
        (c.tlhip_gemv_mxfp4_rmsnorm_gateup, (p, None, p, None, p, p, p, 2, 33, 1e-6), EINVAL),
        (c.tlhip_gemm_mxfp4_nt, (p, None, p, p, p, 1, 1, 32), EINVAL), (c.tlhip_gemm_mxfp4_nt, (p, p, p, p, p, 0, 1, 32), EINVAL),
        (c.tlhip_gemm_mxfp4_nt, (p, p, p, p, p, 1, 1, 31), EINVAL), (c.tlhip_gemm_mxfp4_nt, (odd, p, p, p, p, 1, 1, 32), EINVAL),
        (c.tlhip_gemm_mxfp4_nt, (p, p, p, p, p, 1 << 30, 1, 32), EUNSUPPORTED),
        (c.tlhip_gemm_mxfp4_nt_parts, (p, p, p, p, p, 255, 2, 32, 32, C.byref(n)), EINVAL),
        (c.tlhip_gemm_mxfp4_nt_parts, (p, p, p, p, p, 256, 2, 32, 32, None), EINVAL),
        (c.tlhip_gemm_mxfp4_nt_swiglu, (p, p, p, p, p, p, 1, 33, 32), EINVAL),
        (c.tlhip_gemm_mxfp4_nt_swiglu, (p, p, p, p, p, None, 1, 32, 32), EINVAL),
        (c.tlhip_gemm_mxfp4_nt_swiglu, (p, p, p, p, odd, p, 1, 32, 32), EINVAL),
    ]
    q, t, u = p + 4096, p + 8192, p + 12288      # written over what is read
    cases += [
        (c.tlhip_quantize_mxfp4, (p, 0, p, t, 1, 32), EINVAL), (c.tlhip_quantize_mxfp4, (p, 0, q, q, 1, 32), EINVAL),
        (c.tlhip_quantize_mxfp8, (p, p, t, 1, 32), EINVAL), (c.tlhip_quantize_mxfp8, (p, q, p, 1, 32), EINVAL),
        (c.tlhip_dequantize_mxfp4, (p, q, p, 0, 1, 32), EINVAL), (c.tlhip_dequantize_mxfp8, (p, q, q, 0, 1, 32), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, q, None, p, t, 32, 1e-6, 1), EINVAL), (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, q, None, q, t, 32, 1e-6, 1), EINVAL),
        (c.tlhip_rmsnorm_res_mxfp8, (p, q, 1, t, p, q, u, 32, 1e-6, 1), EINVAL), (c.tlhip_rmsnorm_res_mxfp8, (p, None, 0, q, p, t, p, 32, 1e-6, 1), EINVAL),
        (c.tlhip_gemm_mxfp4_nt_swiglu, (p, q, t, u, p, u + 64, 1, 32, 32), EINVAL), (c.tlhip_gemm_mxfp4_nt_swiglu, (p, q, t, u, u + 64, q, 1, 32, 32), EINVAL),
    ]
    before = lib.census()
    for fn, args, want in cases:
        assert fn(*args) == want, (fn.__name__, args)
        assert lib.last_error().startswith(fn.__name__)
    assert lib.census() == before
