"""Every kernel form that a product over MXFP4 weights can take, against 64 bits: the decode products in the vector unit, in blocks
of tiles and in blocks that walk the tiles, each with its numbers of wavefronts; the prompt products in blocks of 16 rows and in
every size of tile. Which form a size takes is asked of the library; the sizes here are held to take all of them.

A large weight's rows repeat a prime number of rows, so that 64 bits are quick and a row in another's place is seen. The bounds are
those of test_gpu_mxfp.py, derived there."""
import importlib
import math
import random

import numpy as np
import pytest

import mx_oracle as mx
from test_gpu_mxfp import EPS, activations, check_gated, guarded, product_bound, rng, rows8, taken, upload_rows, weight

PLAIN, NORMED, MERGED = 0, 1, 2
VECTOR, WALK, TILES = 0, 1, 2


@pytest.fixture(scope="module")
def plans(pkg):
    return pkg.TlHip(init=False)


def row_form(plans, N, K, producer, gated):
    """A form and how many wavefronts share a row in it; in the vector unit that is only a loop's length."""
    form, rows, share, waves, units = plans.plan_gemv_mxfp4(N, K, producer, gated)
    return (producer, gated, form, rows) + ((share, waves, units) if form != VECTOR else ())


def product_form(plans, M, N, K, gated):
    rows, features, tokens, parts, apart = plans.plan_gemm_mxfp4(M, N, K, gated)
    if rows:
        return (gated, True, features, (K > 256) + (K > 512) + (K > 1024), apart)
    return (gated, False, features, tokens, parts > 1, K % 128 == 0, apart)


# rows of the weight (gated: gate rows), K; what is behind the last whole tile is part of one
PLAIN_SHAPES = [(1, 512), (897, 4864), (131408, 32), (66800, 288), (34320, 544), (16432, 1280), (8784, 3584), (16400, 2080), (70, 64), (70, 288), (4300, 33856),
                (1671, 12576), (4113, 32), (4109, 288), (16421, 544), (11729, 1792), (4979, 4224), (3584, 18944)]
NORMED_SHAPES = [(3, 512), (1060, 512), (131408, 32), (66800, 288), (34320, 544), (16496, 1088), (8784, 3584), (151936, 896), (37, 64), (37, 288), (3437, 2752),
                 (21, 33184), (4113, 32), (4109, 288), (12830, 736), (5187, 1824), (4291, 3104), (4608, 3584)]
GATED_SHAPES = [(3, 512), (545, 512), (65680, 32), (34160, 288), (16416, 544), (9456, 1088), (4464, 3328), (18944, 3584), (37, 64), (37, 288), (1873, 2560),
                (21, 33184), (2051, 32), (2115, 288), (7377, 640), (2545, 1856), (2081, 3328)]
# rows, heads, head size, splits
MERGED_SHAPES = [(5, 8, 64, 4), (1060, 4, 128, 3), (30, 2, 64, 16), (30, 6, 64, 5), (3219, 23, 128, 8), (21, 260, 128, 7), (4113, 1, 128, 2), (4130, 6, 64, 9), (9555, 8, 128, 8),
                 (4109, 36, 64, 16), (4306, 25, 128, 2)]
# M, N (gated: gate rows), K, gated
PRODUCT_SHAPES = [(65, 99, 96, False), (65, 4131, 384, False), (65, 4131, 2080, False), (65, 2082, 4224, False), (131, 16421, 96, False), (131, 16418, 384, False),
                  (67, 8226, 4224, False), (1003, 5155, 96, False), (1003, 5157, 384, False), (65, 99, 160, False), (65, 99, 384, False), (65, 99, 992, False), (65, 99, 1120, False),
                  (701, 99, 160, False), (701, 99, 384, False), (301, 515, 928, False), (301, 515, 1120, False), (5, 8395, 13376, False), (65, 12845, 5600, False),
                  (67, 18391, 5632, False), (1423, 22519, 96, False), (2066, 15795, 128, False),
                  (65, 96, 96, True), (65, 96, 384, True), (65, 96, 2080, True), (65, 96, 2176, True), (67, 12320, 96, True), (67, 12320, 384, True), (67, 4128, 4224, True),
                  (203, 12320, 96, True), (203, 12320, 384, True), (1501, 12320, 96, True), (1501, 12320, 384, True), (65, 96, 1120, True), (131, 288, 1120, True),
                  (9, 96, 160, True), (9, 96, 384, True), (9, 96, 992, True), (9, 4608, 1120, True), (2, 2112, 5728, True),
                  (67, 6144, 5056, True), (66, 4960, 5632, True), (503, 64, 928, True)]


def _draw(r, lo, hi):
    return int(round(lo * (hi / lo) ** r.random()))


def test_every_form_of_the_decode_products_is_among_the_sizes(plans):
    have = {row_form(plans, N, K, PLAIN, False) for N, K in PLAIN_SHAPES} | {row_form(plans, N, K, NORMED, False) for N, K in NORMED_SHAPES}
    have |= {row_form(plans, N, K, NORMED, True) for N, K in GATED_SHAPES} | {row_form(plans, N, h * D, MERGED, False) for N, h, D, _ in MERGED_SHAPES}
    r, missing = random.Random(1), {}
    for _ in range(30000):
        N, K = _draw(r, 1, 1 << 18), 32 * _draw(r, 1, 2048)
        N = N if r.random() < 0.4 else -(-N // 16) * 16
        for producer, gated in ((PLAIN, False), (NORMED, False), (NORMED, True), (MERGED, False)):
            k = max(64, K // 64 * 64) if producer == MERGED else K
            form = row_form(plans, N, k, producer, gated)
            if form not in have:
                missing.setdefault(form, (N, k))
    assert not missing


def test_every_form_of_the_prompt_products_is_among_the_sizes(plans):
    have = {product_form(plans, *s) for s in PRODUCT_SHAPES}
    r, missing = random.Random(2), {}
    for _ in range(30000):
        M, N, K, gated = _draw(r, 1, 1 << 12), _draw(r, 1, 1 << 15), 32 * _draw(r, 1, 592), r.random() < 0.5
        N = -(-N // 32) * 32 if gated else N
        form = product_form(plans, M, N, K, gated)
        if form not in have:
            missing.setdefault(form, (M, N, K))
    assert not missing


def test_products_of_the_largest_results_have_tiles_enough(plans):
    """Every size that is not refused is in fewer than 2^24 tiles, blocks of 256 threads that a grid counts in 32 bits."""
    r = random.Random(3)
    cases = [(1 << 20, 1 << 17, True), (1 << 20, 65568, True), (1 << 13, 1 << 24, True), (8191, 1 << 24, True), (1 << 20, (1 << 17) - 32, True)]
    for _ in range(4000):
        M = _draw(r, 1 << 12, 1 << 20)
        cases.append((M, max(32, min(1 << 24, (1 << 37) // M) // 32 * 32 - 32 * r.randint(0, 3)), r.random() < 0.7))
    for M, N, gated in cases:
        rows, features, tokens, _, _ = plans.plan_gemm_mxfp4(M, N, 32 * r.randint(1, 3), gated)
        assert rows or -(-N // (features // 2 if gated else features)) * -(-M // tokens) < 1 << 24, (M, N, gated)


PERIOD = 257


def repeated(r, n, k, seed=0):
    """A weight of n rows that repeat, and the rows that they repeat: codes, scales, values"""
    codes, scales = weight(r, min(n, PERIOD), k)
    at = np.arange(n) % PERIOD
    return codes[at], scales[at], mx.values(codes, scales, True)


def spread(base, n):
    return base[..., np.arange(n) % PERIOD]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", PLAIN_SHAPES)
def test_token_product(lib, N, K):
    r = rng(101, N, K)
    x, (wc, wsc, w) = activations(r, 1, K), repeated(r, N, K)
    bufs, dx, out = upload_rows(lib, wc, wsc, True), lib.to_device(x), guarded(lib, 4 * N)
    lib.gemv_mxfp4(dx, *bufs, out, N, K)
    x64 = x[0].astype(np.float64)
    big = np.abs(x64).reshape(-1, 32).max(-1).repeat(32)
    bound = product_bound(x64[None], w, K)[0] + 2.0 ** -38 * (np.abs(w) @ big)
    assert (np.abs(taken(out, 4 * N, np.float32, (N,)) - spread(w @ x64, N)) <= spread(bound, N)).all()
    for b in bufs + (dx, out):
        b.free()


def normed_row(r, K, delta):
    x, d, nw = activations(r, 1, K)[0], activations(r, 1, K)[0], (1 + 0.1 * r.standard_normal(K)).astype(np.float32)
    s = x + d if delta else x
    s64 = s.astype(np.float64)
    return x, d if delta else None, nw, s, s64 / np.sqrt((s64 * s64).mean() + EPS) * nw


def norm_rel(K):
    return (K / 64 + 20) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", NORMED_SHAPES)
@pytest.mark.parametrize("delta", [False, True])
def test_token_product_behind_a_norm(lib, N, K, delta):
    r = rng(102, N, K)
    (x, d, nw, s, h), (wc, wsc, w) = normed_row(r, K, delta), repeated(r, N, K)
    bufs = upload_rows(lib, wc, wsc, True) + tuple(lib.to_device(a) for a in (x, nw) + ((d,) if delta else ()))
    out, xout = guarded(lib, 4 * N), guarded(lib, 4 * K)
    lib.gemv_mxfp4_rmsnorm(bufs[2], bufs[4] if delta else None, bufs[3], xout, *bufs[:2], out, N, K, EPS)
    assert np.array_equal(taken(xout, 4 * K, np.float32, (K,)), s)
    bound = product_bound(h[None], w, K)[0] + norm_rel(K) * (np.abs(w) @ np.abs(h))
    assert (np.abs(taken(out, 4 * N, np.float32, (N,)) - spread(w @ h, N)) <= spread(bound, N)).all()
    for b in bufs + (out, xout):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("ff,K", GATED_SHAPES)
@pytest.mark.parametrize("delta", [False, True])
def test_gated_token_product_behind_a_norm(lib, ff, K, delta):
    r = rng(103, ff, K)
    (x, d, nw, s, h), (gc, gs, wg), (uc, us, wu) = normed_row(r, K, delta), repeated(r, ff, K), repeated(r, ff, K)
    bufs = upload_rows(lib, np.concatenate([gc, uc]), np.concatenate([gs, us]), True) + tuple(lib.to_device(a) for a in (x, nw) + ((d,) if delta else ()))
    out, xout = guarded(lib, 4 * ff), guarded(lib, 4 * K)
    lib.gemv_mxfp4_rmsnorm_gateup(bufs[2], bufs[4] if delta else None, bufs[3], xout, *bufs[:2], out, 2 * ff, K, EPS)
    assert np.array_equal(taken(xout, 4 * K, np.float32, (K,)), s)
    g, u = wg @ h, wu @ h
    og, ou = (product_bound(h[None], w, K)[0] + norm_rel(K) * (np.abs(w) @ np.abs(h)) for w in (wg, wu))
    silu = g / (1 + np.exp(-g))
    off = 1.1 * np.abs(u) * og + np.abs(silu) * ou + 1.2 * og * ou + np.abs(silu * u) * 2.0 ** -20 + 1e-37
    assert (np.abs(taken(out, 4 * ff, np.float32, (ff,)) - spread(silu * u, ff)) <= spread(off, ff)).all()
    for b in bufs + (out, xout):
        b.free()


def splits(r, heads, D, S):
    m = r.uniform(-30, 30, (heads, S)).astype(np.float32)
    l = r.uniform(0.5, 64, (heads, S)).astype(np.float32)
    return m, l, (r.standard_normal((heads, S, D)) * l[:, :, None]).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("N,heads,D,S", MERGED_SHAPES)
def test_token_product_of_the_attentions_splits(lib, N, heads, D, S):
    r, K = rng(104, N, heads, D), heads * D
    (m, l, acc), (wc, wsc, w) = splits(r, heads, D, S), repeated(r, N, K)
    bufs = upload_rows(lib, wc, wsc, True) + (lib.to_device(np.concatenate([m.ravel(), l.ravel(), acc.ravel()])),)
    out = guarded(lib, 4 * N)
    lib.gemv_mxfp4_attn(bufs[2], S, heads, D, *bufs[:2], out, N, K)
    e = np.exp(m.astype(np.float64) - m.max(axis=1, keepdims=True))
    row, size = (((e[:, :, None] * a).sum(axis=1) / (e * l).sum(axis=1)[:, None]).reshape(K) for a in (acc, np.abs(acc)))
    bound = (128 + K / 128 + 64 + 2 * (60 / np.log(2) + 4 + S) + 1) * 2.0 ** -24 * (np.abs(w) @ size)
    assert (np.abs(taken(out, 4 * N, np.float32, (N,)) - spread(w @ row, N)) <= spread(bound, N)).all()
    for b in bufs + (out,):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,gated", PRODUCT_SHAPES)
def test_prompt_product(lib, M, N, K, gated):
    r = rng(105, M, N, K)
    (ac, asc), (wc, wsc, w) = rows8(r, M, K), repeated(r, N, K)
    a = mx.values(ac, asc, False)
    if not gated:
        bufs, out = upload_rows(lib, ac, asc) + upload_rows(lib, wc, wsc, True), guarded(lib, 4 * M * N)
        lib.gemm_mxfp4_nt(*bufs, out, M, N, K)
        got = taken(out, 4 * M * N, np.float32, (M, N))
        want, bound = a @ w.T, product_bound(a, w, K)
        for n in range(0, N, PERIOD):
            c = min(PERIOD, N - n)
            assert (np.abs(got[:, n:n + c] - want[:, :c]) <= bound[:, :c]).all(), n
        freed = bufs + (out,)
    else:
        uc, us, wu = repeated(r, N, K)
        wsc, us = (wsc + 3).astype(np.uint8), (us + 3).astype(np.uint8)
        bufs = upload_rows(lib, ac, asc) + upload_rows(lib, np.concatenate([wc, uc]), np.concatenate([wsc, us]), True)
        codes, scales = guarded(lib, M * N), guarded(lib, M * N // 32)
        lib.gemm_mxfp4_nt_swiglu(*bufs, codes, scales, M, N, K)
        got_c, got_s = taken(codes, M * N, np.uint8, (M, N)), taken(scales, M * N // 32, np.uint8, (M, N // 32))
        wg, wu, step = mx.values(wc[:PERIOD], wsc[:PERIOD], True), mx.values(uc[:PERIOD], us[:PERIOD], True), 32 * 64
        for n in range(0, N, step):               # (features in pieces, whole blocks of them)
            at = np.arange(n, min(n + step, N)) % PERIOD
            check_gated(got_c[:, n:n + step], got_s[:, n // 32:(n + step) // 32], a, np.concatenate([wg[at], wu[at]]), K)
        freed = bufs + (codes, scales)
    for b in freed:
        b.free()


# the row's digits in blocks of tiles, of 16 and of 32 rows, and in blocks that walk them; and the vector unit
HARD = [(70, 288), (4128, 480), (1671, 12576), (34320, 544), (16432, 1280), (8784, 3584), (897, 4864)]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", HARD)
@pytest.mark.parametrize("kind", ["spread", "largest", "top", "smallest", "bottom", "results at the bottom", "one outlier", "blocks apart"])
def test_token_product_of_hard_rows(lib, N, K, kind):
    """f32 sums of the row's numbers as they are: magnitudes all over a block, or over the row's blocks, at both ends of f32, and one
    that dwarfs its neighbours under weights of zero. Twelve digits' sums of y / 256 have 192 + K / 128 roundings each, of 2^-150 where
    they are subnormal."""
    r = rng(106, N, K)
    x, (wc, wsc) = r.standard_normal((1, K)).astype(np.float32), weight(r, min(N, PERIOD), K)
    if kind == "spread":
        x *= 2.0 ** r.integers(-22, 1, (1, K)).astype(np.float32)
    elif kind == "largest":
        x *= np.float32(2.0 ** 125) / np.abs(x).max()
        wsc = (wsc - 8).astype(np.uint8)
    elif kind == "top":                                    # (exponent fields 253 and 254 among the blocks' largest)
        x *= np.float32(3.3e38) / np.abs(x).reshape(-1, 32).max(-1).repeat(32)
        x[0, 32:64] *= np.float32(0.4)
        wsc = (wsc - 24).astype(np.uint8)
    elif kind == "smallest":
        x *= np.float32(2.0 ** -100)
        wsc = (wsc + 20).astype(np.uint8)
    elif kind == "bottom":                                 # (largest numbers of 2^-78 to 2^-148)
        x = (x / np.abs(x).max() * 2.0 ** -r.integers(78, 149, K // 32).astype(np.float64).repeat(32)).astype(np.float32)
        wsc = (wsc + 60).astype(np.uint8)
    elif kind == "results at the bottom":                  # (some of them subnormal)
        x *= np.float32(2.0 ** -66)
        wsc = (wsc - 66).astype(np.uint8)
    elif kind == "one outlier":
        x[0, 5::32] = 2.0 ** 20
        wc[:, 5::32] &= 8
    else:
        x = (x * 2.0 ** r.integers(-40, 41, K // 32).astype(np.float64).repeat(32)).astype(np.float32)
    at = np.arange(N) % PERIOD
    w, x64 = mx.values(wc, wsc, True), x[0].astype(np.float64)
    bufs, dx, out = upload_rows(lib, wc[at], wsc[at], True), lib.to_device(x), guarded(lib, 4 * N)
    lib.gemv_mxfp4(dx, *bufs, out, N, K)
    big = np.abs(x64).reshape(-1, 32).max(-1).repeat(32)
    bound = product_bound(x64[None], w, K)[0] + np.abs(w) @ np.maximum(2.0 ** -48 * big, 2.0 ** -128) + 12 * (192 + K / 128) * 2.0 ** -142
    assert (np.abs(taken(out, 4 * N, np.float32, (N,)) - spread(w @ x64, N)) <= spread(bound, N)).all()
    for b in bufs + (dx, out):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", HARD)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_token_product_of_small_and_large_numbers(lib, N, K, scale):
    r = rng(107, N, K)
    x, (wc, wsc, w) = activations(r, 1, K) * np.float32(scale), repeated(r, N, K)
    bufs, dx, out = upload_rows(lib, wc, wsc, True), lib.to_device(x), guarded(lib, 4 * N)
    lib.gemv_mxfp4(dx, *bufs, out, N, K)
    x64 = x[0].astype(np.float64)
    big = np.abs(x64).reshape(-1, 32).max(-1).repeat(32)
    bound = product_bound(x64[None], w, K)[0] + 2.0 ** -38 * (np.abs(w) @ big)
    assert (np.abs(taken(out, 4 * N, np.float32, (N,)) - spread(w @ x64, N)) <= spread(bound, N)).all()
    for b in bufs + (dx, out):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", HARD + [(4464, 3328), (2081, 3328), (1060, 512)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_rows_and_weights_that_are_not_finite(lib, N, K, bad):
    """A number of the row that is not finite makes every result NaN, wherever it is and whichever operand of the sum it comes in with;
    a block of the weight with scale 255 its own row's alone."""
    r = rng(108, N, K)
    x, nw, (wc, wsc, _) = activations(r, 1, K)[0], np.ones(K, np.float32), repeated(r, 2 * N, K)
    zero = lib.to_device(np.zeros(K, np.float32))
    bufs, dnw, out, act = upload_rows(lib, wc, wsc, True), lib.to_device(nw), lib.empty(N), lib.empty(N)
    for k in (0, K // 2 + 1, K - 1):
        worse = x.copy()
        worse[k] = bad
        dx, dy = lib.to_device(worse), lib.to_device(x)
        lib.gemv_mxfp4(dx, *bufs, out, N, K)
        assert np.isnan(out.numpy()).all(), k
        for a, d in ((dx, None), (dx, zero), (dy, dx)):
            lib.gemv_mxfp4_rmsnorm(a, d, dnw, None, *bufs, out, N, K, EPS)
            lib.gemv_mxfp4_rmsnorm_gateup(a, d, dnw, None, *bufs, act, 2 * N, K, EPS)
            assert np.isnan(out.numpy()).all() and np.isnan(act.numpy()).all(), k
        dx.free()
        dy.free()
    lib.gemv_mxfp4_rmsnorm(zero, None, dnw, None, *bufs, out, N, K, EPS)
    assert not out.numpy().any()
    wsc[0, -1] = wsc[N - 1, 0] = wsc[N // 2, K // 64] = wsc[2 * N - 1, -1] = 255
    worse = upload_rows(lib, wc, wsc, True)
    lib.gemv_mxfp4_rmsnorm(zero, None, dnw, None, *worse, out, N, K, EPS)
    lib.gemv_mxfp4_rmsnorm_gateup(zero, None, dnw, None, *worse, act, 2 * N, K, EPS)
    rows = np.isin(np.arange(N), [0, N // 2, N - 1])
    assert np.array_equal(np.isnan(out.numpy()), rows) and np.array_equal(np.isnan(act.numpy()), rows)
    dx = lib.to_device(x)
    lib.gemv_mxfp4(dx, *worse, out, N, K)
    assert np.array_equal(np.isnan(out.numpy()), rows)
    for b in bufs + worse + (zero, dnw, out, act, dx):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("N,heads,D,S", [(5, 8, 64, 4), (30, 2, 64, 16), (4306, 25, 128, 2)])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_splits_that_are_not_finite(lib, N, heads, D, S, bad):
    r, K = rng(109, N), heads * D
    m, l, acc = splits(r, heads, D, S)
    m[:] = r.uniform(-1, 1, m.shape)
    acc[heads - 1, S - 1, D - 1] = bad
    wc, wsc, _ = repeated(r, N, K)
    bufs, out = upload_rows(lib, wc, wsc, True) + (lib.to_device(np.concatenate([m.ravel(), l.ravel(), acc.ravel()])),), lib.empty(N)
    lib.gemv_mxfp4_attn(bufs[2], S, heads, D, *bufs[:2], out, N, K)
    assert np.isnan(out.numpy()).all()
    for b in bufs + (out,):
        b.free()
