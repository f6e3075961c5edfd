"""Products over MXFP4 weights whose results lie where, or are as large as, no ordinary ones: rows of logits behind one another at any
multiple of four bytes, results of more than 2^36 numbers, weights of more than one launch of the rounding."""
import importlib

import numpy as np
import pytest

import mx_oracle as mx
from test_gpu_gguf import SMALL, WIDE_HEAD, synth_weights
from test_gpu_mxfp import activations, check_gated, product_bound, rng, rows8, upload_rows, weight
from test_gpu_mxfp_model import opened, tokens_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims,vocab", [(SMALL, 1001), (SMALL, 1002), (WIDE_HEAD, 323)])
def test_logits_of_several_rows_of_any_vocabulary(tmp_path, dims, vocab):
    """Rows of logits that no 16 bytes divide: each is what it is when it is asked for alone."""
    model = importlib.import_module("cpp-tensorlib_amd.model")
    d = dict(dims, vocab=vocab)
    path, ids, want = opened(tmp_path, d, synth_weights(d, seed=31)), tokens_of(d, 30, 37), [0, 7, 8, 29]
    m = model.Model.open(path, max_ctx=d["max_ctx"], mxfp4=True)
    many = m.feed(ids, want=want)
    assert many.shape == (4, vocab)
    for i, t in enumerate(want):
        m.reset()
        assert np.array_equal(m.feed(ids, want=[t])[0], many[i])
    m.close()


# a row of the weight in the vector unit, in tiles of 16, in blocks that walk the tiles
@pytest.mark.parametrize("N,K", [(5, 896), (35, 160), (16640, 2048)])
@pytest.mark.parametrize("off", [4, 8, 12])
def test_results_at_any_number(lib, N, K, off):
    r = rng(41, N, K)
    x, (wc, wsc) = activations(r, 1, K), weight(r, N, K)
    bufs, out, dx, nw = upload_rows(lib, wc, wsc, True), lib.empty_bytes(4 * N + 32), lib.to_device(x), lib.to_device(np.ones(K, np.float32))
    w, x64 = mx.values(wc, wsc, True), x[0].astype(np.float64)
    big = np.abs(x64).reshape(-1, 32).max(-1).repeat(32)
    h = x64 / np.sqrt((x64 * x64).mean() + 1e-6)
    plain = w @ x64, product_bound(x64[None], w, K)[0] + 2.0 ** -38 * (np.abs(w) @ big)
    normed = w @ h, product_bound(h[None], w, K)[0] + (K / 64 + 20) * 2.0 ** -24 * (np.abs(w) @ np.abs(h))
    for call, (want, bound) in ((lambda: lib.gemv_mxfp4(dx, *bufs, out, N, K), plain),
                                (lambda: lib.gemv_mxfp4_rmsnorm(dx, None, nw, None, *bufs, out, N, K, 1e-6), normed)):
        lib._chk(lib.c.tlhip_fill_u32(out.ptr, 0xa5a5a5a5, N + 8))
        out.ptr += off
        call()
        out.ptr -= off
        got = out.numpy(np.uint8)
        assert (got[:off] == 0xa5).all() and (got[off + 4 * N:] == 0xa5).all(), "wrote beside the result"
        assert (np.abs(got[off:off + 4 * N].copy().view(np.float32) - want) <= bound).all()
    for b in bufs + (out, dx, nw):
        b.free()


def test_gated_result_of_more_than_2_to_the_36_numbers(lib):
    """64 GB of elements, in more than 2^22 tiles; rows from all over it, the first and the last, against 64 bits."""
    r, M, ff, K = rng(43), 1 << 20, 65568, 32
    (ac, asc), (wc, wsc) = rows8(r, M, K), weight(r, 2 * ff, K)
    wsc = (wsc + 3).astype(np.uint8)
    bufs = upload_rows(lib, ac, asc) + upload_rows(lib, wc, wsc, True)
    codes, scales = lib.empty_bytes(M * ff + 256), lib.empty_bytes(M * ff // 32 + 256)
    for b, n in ((codes, M * ff), (scales, M * ff // 32)):
        lib._chk(lib.c.tlhip_fill_u32(b.ptr + n, 0xa5a5a5a5, 64))
    lib.gemm_mxfp4_nt_swiglu(*bufs, codes, scales, M, ff, K)

    def read(ptr, n):
        out = np.empty(n, np.uint8)
        lib._chk(lib.c.tlhip_memcpy_d2h(out.ctypes.data, ptr, n))
        return out

    rows = np.unique(np.concatenate([[0, 1, 127, 128, M // 2 - 1, M // 2, M - 129, M - 128, M - 2, M - 1], r.integers(0, M, 8)]))
    got_c = np.stack([read(codes.ptr + int(m) * ff, ff) for m in rows])
    got_s = np.stack([read(scales.ptr + int(m) * (ff // 32), ff // 32) for m in rows])
    check_gated(got_c, got_s, mx.values(ac[rows], asc[rows], False), mx.values(wc, wsc, True), K)
    assert (read(codes.ptr + M * ff, 256) == 0xa5).all() and (read(scales.ptr + M * ff // 32, 256) == 0xa5).all(), "wrote behind the result"
    for b in bufs + (codes, scales):
        b.free()


def test_rounding_of_more_than_one_launch(lib):
    """More than 2^34 numbers, 2^31 lanes of eight, which a grid counts: ones, but random rows at the first launch's end and at the last."""
    r, K = rng(47), 65536
    rows = (1 << 18) + 40
    src, codes, scales = lib.empty_bytes(rows * K * 2), lib.empty_bytes(rows * K // 2), lib.empty_bytes(rows * K // 32)
    lib._chk(lib.c.tlhip_fill_u32(src.ptr, 0x3f803f80, rows * K // 2))
    x = (r.standard_normal((70, K)).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    at = np.concatenate([np.arange((1 << 18) - 30, (1 << 18) + 30), np.arange(rows - 10, rows)])
    for ptr, a in ((src.ptr + int(at[0]) * K * 2, x[:60]), (src.ptr + int(at[60]) * K * 2, x[60:])):
        a = np.ascontiguousarray(a)
        lib._chk(lib.c.tlhip_memcpy_h2d(ptr, a.ctypes.data, a.nbytes))
    lib.quantize_mxfp4(src, lib.T_BF16, codes, scales, rows, K)
    lib.dequantize_mxfp4(codes, scales, src, lib.T_BF16, rows, K)
    want_c, want_s = mx.quantize((x.astype(np.uint32) << 16).view(np.float32), True)
    want = mx.values(want_c, want_s, True)

    def read(b, row, each, dtype):
        out = np.empty(each, dtype)
        lib._chk(lib.c.tlhip_memcpy_d2h(out.ctypes.data, b.ptr + int(row) * out.nbytes, out.nbytes))
        return out

    for i, row in enumerate(at):
        assert np.array_equal(read(codes, row, K // 2, np.uint8), mx.pack(want_c[i:i + 1])[0]), row
        assert np.array_equal(read(scales, row, K // 32, np.uint8), want_s[i]), row
        assert np.array_equal((read(src, row, K, np.uint16).astype(np.uint32) << 16).view(np.float32), want[i].astype(np.float32)), row
    for row in (0, 12345, at[0] - 1, at[59] + 1 if at[59] + 1 < at[60] else 1):       # 1 = 4 x 2^-2
        assert (read(codes, row, K // 2, np.uint8) == 0x66).all() and (read(scales, row, K // 32, np.uint8) == 125).all()
        assert (read(src, row, K, np.uint16) == 0x3f80).all()
    for b in (src, codes, scales):
        b.free()
