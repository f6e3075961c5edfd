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


@pytest.mark.parametrize("result,operand", [(4, 3), (5, 3), (6, 3), (4, 1), (5, 1), (6, 1), (5, 0), (6, 0), (5, 4), (6, 4), (6, 5)])
def test_norm_over_its_operands_is_refused(refused, at, result, operand):
    """A row's block writes what the blocks of other rows still read: the weights, the parts, another row's result."""
    args = [at[0], at[1], 2, at[2], at[3], at[4], at[5], 64, 1e-6, 3]      # x, parts, S, w, xout, codes, scales, n, eps, rows
    args[result] = args[operand]
    refused("tlhip_rmsnorm_res_mxfp8", args, EINVAL, "must not be")


def test_norm_in_place_of_a_row_that_is_also_the_weights_is_refused(refused, at):
    refused("tlhip_rmsnorm_res_mxfp8", (at[0], at[1], 2, at[0], at[0], at[4], at[5], 64, 1e-6, 3), EINVAL, "must not be")
    refused("tlhip_rmsnorm_res_mxfp8", (at[0], at[0], 2, at[1], at[0], at[4], at[5], 64, 1e-6, 3), EINVAL, "must not be")
