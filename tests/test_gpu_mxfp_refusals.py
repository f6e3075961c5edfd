"""What the microscaled formats' entry points refuse, one reason at a time: every call here would be a good one but for the one
thing that its case names, and its pointers are apart from each other unless that is the case."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
EINVAL, EUNSUPPORTED = -2, -3


@pytest.fixture
def refused(lib):
    """refused(entry, arguments, code, words): the call gives the code, tells these words behind its name, and launches nothing."""
    def check(entry, args, code, words):
        before = lib.census()
        assert getattr(lib.c, entry)(*args) == code, (entry, args, lib.last_error())
        told = lib.last_error()
        assert told.startswith(entry + ": ") and words in told, told
        assert lib.census() == before
    return check


@pytest.fixture
def at(lib):
    """Eight places of 64 KB in one buffer"""
    b = lib.empty_bytes(8 << 16)
    yield [b.ptr + (i << 16) for i in range(8)]
    b.free()


GOOD = {                      # arguments of a small call of each, numbers for the places that `at` gives
    "tlhip_quantize_mxfp4": ("p0", 0, "p1", "p2", 3, 64),
    "tlhip_quantize_mxfp8": ("p0", "p1", "p2", 3, 64),
    "tlhip_dequantize_mxfp4": ("p0", "p1", "p2", 0, 3, 64),
    "tlhip_dequantize_mxfp8": ("p0", "p1", "p2", 2, 3, 64),
    "tlhip_rmsnorm_res_mxfp8": ("p0", "p1", 2, "p2", "p3", "p4", "p5", 64, 1e-6, 3),
    "tlhip_gemv_mxfp4": ("p0", "p1", "p2", "p3", 5, 64),
    "tlhip_gemv_mxfp4_attn": ("p0", 2, 2, 64, "p1", "p2", "p3", 5, 128),
    "tlhip_gemv_mxfp4_rmsnorm": ("p0", "p1", "p2", "p3", "p4", "p5", "p6", 5, 64, 1e-6),
    "tlhip_gemv_mxfp4_rmsnorm_gateup": ("p0", "p1", "p2", "p3", "p4", "p5", "p6", 10, 64, 1e-6),
    "tlhip_gemm_mxfp4_nt": ("p0", "p1", "p2", "p3", "p4", 3, 5, 64),
    "tlhip_gemm_mxfp4_nt_parts": ("p0", "p1", "p2", "p3", "p4", 60, 3, 5, 64, "count"),
    "tlhip_gemm_mxfp4_nt_swiglu": ("p0", "p1", "p2", "p3", "p4", "p5", 3, 32, 64),
}
QUANTIZE = [(EINVAL, "rows > 0", "rows", (0, -1, -(1 << 62))), (EINVAL, "multiple of 32", "K", (0, -32, 16, 33, 65, 1 << 31 | 1)),
            (EUNSUPPORTED, "too many", "rows", (1 << 60,))]
PRODUCT = [(EINVAL, "M, N > 0", "N", (0, -1)), (EINVAL, "multiple of 32", "K", (0, -32, 16, 33, 72))]
# entry, {name of an argument: its place}, what is refused of which argument: (code, words, name, values); "odd": its place and 4
# bytes, "odder": and 2
CASES = [
    ("tlhip_quantize_mxfp4", dict(src=0, type=1, codes=2, scales=3, rows=4, K=5), QUANTIZE + [
        (EINVAL, "null pointer", ("src", "codes", "scales"), (None,)), (EUNSUPPORTED, "element type", "type", (3, -1, 99)),
        (EINVAL, "16-byte aligned", ("src", "codes"), ("odd",))]),
    ("tlhip_quantize_mxfp8", dict(x=0, codes=1, scales=2, rows=3, K=4), QUANTIZE + [
        (EINVAL, "null pointer", ("x", "codes", "scales"), (None,)), (EINVAL, "16-byte aligned", ("x", "codes"), ("odd",))]),
    ("tlhip_dequantize_mxfp4", dict(codes=0, scales=1, dst=2, type=3, rows=4, K=5), QUANTIZE + [
        (EINVAL, "null pointer", ("codes", "scales", "dst"), (None,)), (EUNSUPPORTED, "element type", "type", (1, 3, -1)),
        (EINVAL, "16-byte aligned", ("codes", "dst"), ("odd",))]),
    ("tlhip_dequantize_mxfp8", dict(codes=0, scales=1, dst=2, type=3, rows=4, K=5), QUANTIZE + [
        (EINVAL, "null pointer", ("codes", "scales", "dst"), (None,)), (EUNSUPPORTED, "element type", "type", (1, 3, -1)),
        (EINVAL, "16-byte aligned", ("codes", "dst"), ("odd",))]),
    ("tlhip_rmsnorm_res_mxfp8", dict(x=0, parts=1, S=2, w=3, xout=4, codes=5, scales=6, n=7, rows=9), [
        (EINVAL, "null pointer", ("x", "parts", "w", "codes", "scales"), (None,)), (EINVAL, "rows > 0", "rows", (0, -1)),
        (EINVAL, "multiple of 32", "n", (0, -32, 16, 40)), (EUNSUPPORTED, "at most 64 parts", "S", (-1, 65, 1 << 40)),
        (EUNSUPPORTED, "rows of 32768", "n", (32800, 1 << 33)), (EUNSUPPORTED, "2^20 rows", "rows", ((1 << 20) + 1, 1 << 40)),
        (EINVAL, "16-byte aligned", ("x", "parts", "w", "xout", "codes"), ("odd",))]),
    ("tlhip_gemv_mxfp4", dict(a=0, codes=1, scales=2, y=3, N=4, K=5), PRODUCT + [
        (EINVAL, "null pointer", ("a", "codes", "scales", "y"), (None,)), (EINVAL, "16-byte aligned", ("a", "codes"), ("odd",)),
        (EINVAL, "4-byte aligned", "y", ("odder",)), (EUNSUPPORTED, "N up to 2^24", "N", ((1 << 24) + 1, 1 << 40)),
        (EUNSUPPORTED, "K up to 65536", "K", (65568, 1 << 40))]),
    ("tlhip_gemv_mxfp4_attn", dict(parts=0, S=1, heads=2, dim=3, codes=4, scales=5, y=6, N=7, K=8), [
        (EINVAL, "M, N > 0", "N", (0, -1)), (EINVAL, "null pointer", ("parts", "codes", "scales", "y"), (None,)),
        (EINVAL, "16-byte aligned", ("parts", "codes"), ("odd",)), (EINVAL, "4-byte aligned", "y", ("odder",)),
        (EUNSUPPORTED, "split partials", "S", (0, -1, 17)), (EINVAL, "heads x head_dim", "heads", (0, -2, 1, 3, 5000)),
        (EINVAL, "heads x head_dim", "dim", (32, 128, 0)), (EINVAL, "heads x head_dim", "K", (64, 160, 256)),
        (EUNSUPPORTED, "N up to 2^24", "N", ((1 << 24) + 1,))]),
    ("tlhip_gemv_mxfp4_rmsnorm", dict(x=0, delta=1, norm_w=2, xout=3, codes=4, scales=5, y=6, N=7, K=8), PRODUCT + [
        (EINVAL, "null pointer", ("x", "norm_w", "codes", "scales", "y"), (None,)),
        (EINVAL, "16-byte aligned", ("x", "delta", "norm_w", "xout", "codes"), ("odd",)), (EINVAL, "4-byte aligned", "y", ("odder",)),
        (EUNSUPPORTED, "N up to 2^24", "N", ((1 << 24) + 1,)), (EUNSUPPORTED, "K up to 65536", "K", (65568,))]),
    ("tlhip_gemv_mxfp4_rmsnorm_gateup", dict(x=0, delta=1, norm_w=2, xout=3, codes=4, scales=5, y=6, N2=7, K=8), [
        (EINVAL, "M, N > 0", "N2", (0, -2)), (EINVAL, "as many gate rows", "N2", (3, 11, -1)), PRODUCT[1],
        (EINVAL, "null pointer", ("x", "norm_w", "codes", "scales", "y"), (None,)),
        (EINVAL, "16-byte aligned", ("x", "delta", "norm_w", "xout", "codes"), ("odd",)), (EINVAL, "4-byte aligned", "y", ("odder",)),
        (EUNSUPPORTED, "N up to 2^24", "N2", ((1 << 25) + 2,)), (EUNSUPPORTED, "K up to 65536", "K", (65568,))]),
    ("tlhip_gemm_mxfp4_nt", dict(ac=0, asc=1, codes=2, scales=3, C=4, M=5, N=6, K=7), PRODUCT + [
        (EINVAL, "M, N > 0", "M", (0, -1)), (EINVAL, "null pointer", ("ac", "asc", "codes", "scales", "C"), (None,)),
        (EINVAL, "16-byte aligned", ("ac", "codes", "C"), ("odd",)), (EUNSUPPORTED, "M up to 2^20", "M", ((1 << 20) + 1, 1 << 40)),
        (EUNSUPPORTED, "N up to 2^24", "N", ((1 << 24) + 1,)), (EUNSUPPORTED, "K up to 65536", "K", (65568,))]),
    ("tlhip_gemm_mxfp4_nt_parts", dict(ac=0, asc=1, codes=2, scales=3, C=4, room=5, M=6, N=7, K=8, n=9), PRODUCT + [
        (EINVAL, "M, N > 0", "M", (0, -1)), (EINVAL, "null pointer", ("ac", "asc", "codes", "scales", "C", "n"), (None,)),
        (EINVAL, "16-byte aligned", ("ac", "codes", "C"), ("odd",)), (EINVAL, "M * N * 4 bytes", "room", (59, 0, -60)),
        (EINVAL, "M * N * 4 bytes", "M", (4, 1 << 20)), (EUNSUPPORTED, "M up to 2^20", "M", ((1 << 20) + 1,)),
        (EUNSUPPORTED, "N up to 2^24", "N", ((1 << 24) + 1,)), (EUNSUPPORTED, "K up to 65536", "K", (65568,))]),
    ("tlhip_gemm_mxfp4_nt_swiglu", dict(ac=0, asc=1, codes=2, scales=3, qc=4, qs=5, M=6, ff=7, K=8), [PRODUCT[1],
        (EINVAL, "M, N > 0", "M", (0, -1)), (EINVAL, "M, N > 0", "ff", (0, -32)), (EINVAL, "ff must be a multiple of 32", "ff", (16, 33, 40)),
        (EINVAL, "null pointer", ("ac", "asc", "codes", "scales", "qc", "qs"), (None,)),
        (EINVAL, "16-byte aligned", ("ac", "codes", "qc"), ("odd",)), (EUNSUPPORTED, "M up to 2^20", "M", ((1 << 20) + 1,)),
        (EUNSUPPORTED, "N up to 2^24", "ff", ((1 << 24) + 32,)), (EUNSUPPORTED, "K up to 65536", "K", (65568,))]),
]
FLAT = [(entry, places[name], code, words, value) for entry, places, refusals in CASES for code, words, names, values in refusals
        for name in ((names,) if isinstance(names, str) else names) for value in values]


@pytest.fixture
def good(at):
    def args(entry):
        count = C.c_int(0)
        return [at[int(a[1:])] if isinstance(a, str) and a != "count" else C.byref(count) if a == "count" else a for a in GOOD[entry]]
    return args


@pytest.mark.parametrize("entry,place,code,words,value", FLAT)
def test_one_bad_argument(refused, good, entry, place, code, words, value):
    args = good(entry)
    args[place] = args[place] + (4 if value == "odd" else 2) if isinstance(value, str) else value
    refused(entry, args, code, words)


@pytest.mark.parametrize("entry", list(GOOD))
def test_the_same_calls_without_it(lib, good, entry):
    """What is refused above is refused for its one argument: the call itself is accepted."""
    assert getattr(lib.c, entry)(*good(entry)) == 0, lib.last_error()
    lib.sync()


def test_results_of_too_many_numbers(refused, good):
    for entry, m, n in (("tlhip_gemm_mxfp4_nt", 5, 6), ("tlhip_gemm_mxfp4_nt_parts", 6, 7), ("tlhip_gemm_mxfp4_nt_swiglu", 6, 7)):
        args = good(entry)
        args[m], args[n] = 1 << 20, (1 << 17) + 32
        refused(entry, args, EUNSUPPORTED, "2^37")


@pytest.mark.parametrize("result,operand", [(4, 3), (5, 3), (6, 3), (4, 1), (5, 1), (6, 1), (5, 0), (6, 0), (5, 4), (6, 4), (6, 5)])
def test_norm_over_its_operands_is_refused(refused, at, result, operand):
    """A row's block writes what the blocks of other rows still read: the weights, the parts, another row's result."""
    args = [at[0], at[1], 2, at[2], at[3], at[4], at[5], 64, 1e-6, 3]      # x, parts, S, w, xout, codes, scales, n, eps, rows
    args[result] = args[operand]
    refused("tlhip_rmsnorm_res_mxfp8", args, EINVAL, "must not be")


def test_norm_in_place_of_a_row_that_is_also_the_weights_is_refused(refused, at):
    refused("tlhip_rmsnorm_res_mxfp8", (at[0], at[1], 2, at[0], at[0], at[4], at[5], 64, 1e-6, 3), EINVAL, "must not be")
    refused("tlhip_rmsnorm_res_mxfp8", (at[0], at[0], 2, at[1], at[0], at[4], at[5], 64, 1e-6, 3), EINVAL, "must not be")
