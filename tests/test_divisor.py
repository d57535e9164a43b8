"""Division by a multiplication (csrc/divisor.hpp, compiled here for the host) against the division.  No GPU needed."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hopper_spmm_amd", "csrc")
SOURCE = """
#include "divisor.hpp"
// how many of n numbers have another quotient than the division's, and the last one of them
extern "C" unsigned wrong(unsigned d, const unsigned *numbers, unsigned n, unsigned *which)
{
    const hspmm::Divisor by = hspmm::Divisor::of(d);
    unsigned count = by.d != d;
    for (unsigned i = 0; i < n; ++i)
        if (by.quotient(numbers[i]) != numbers[i] / d) { ++count; *which = numbers[i]; }
    return count;
}
"""


@pytest.fixture(scope="module")
def divisor(tmp_path_factory):
    at = tmp_path_factory.mktemp("divisor")
    (at / "divisor.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(at / "divisor.so"), str(at / "divisor.cpp")], check=True)
    return ctypes.CDLL(str(at / "divisor.so"))


DIVISORS = list(range(1, 200)) + [x for l in range(8, 31) for x in ((1 << l) - 1, 1 << l, (1 << l) + 1)] + [0x7FFFFFFF, 1000003, 65521, 3 << 28]


@pytest.mark.parametrize("some", range(0, len(DIVISORS), 40))
def test_quotients_are_the_divisions(divisor, some):
    for d in DIVISORS[some:some + 40]:
        # multiples, the numbers beside them, the ends of the range and others
        multiples = d * np.random.default_rng(d).integers(0, 0x7FFFFFFF // d, 3000, endpoint=True)
        n = np.concatenate([multiples, multiples - 1, multiples + d - 1, np.arange(100), 0x7FFFFFFF - np.arange(100), np.random.default_rng(d + 1).integers(0, 1 << 31, 3000)])
        n = np.ascontiguousarray(n[(n >= 0) & (n < 1 << 31)].astype(np.uint32))
        which = ctypes.c_uint()
        assert divisor.wrong(d, n.ctypes.data_as(ctypes.c_void_p), len(n), ctypes.byref(which)) == 0, (d, which.value)
