"""The exact rounding of float32 entries next to the middle of two codes, from the kernels' source on the host, with numbers whose products may be
joined with a sum or difference into one rounding, as a compiler is free to do with plain operators."""
import ctypes
import os
import shutil
import subprocess
from fractions import Fraction

import numpy as np
import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fieldrun_b200", "csrc", "products_8bit.cuh")
SHIMS = """
#include <cmath>
#define __device__
#define __forceinline__ inline

// How a product that is added or subtracted is rounded: 0 by itself, 1 the right operand's joined with the sum, 2 the left one's.
static int joined;

struct Number {
    float v, a = 0, b = 0;             // the value; of a product its factors
    bool product = false;
    Number() = default;
    Number(float v) : v(v) {}
    Number(float a, float b) : v(a * b), a(a), b(b), product(true) {}
    explicit operator int() const { return (int)v; }
    Number operator-() const { return Number(-v); }
    Number operator*(Number o) const { return Number(v, o.v); }
    Number& operator*=(Number o) { return *this = Number(v * o.v); }
    Number operator+(Number o) const {
        if (joined == 1 && o.product) return Number(std::fmaf(o.a, o.b, v));
        if (joined == 2 && product) return Number(std::fmaf(a, b, o.v));
        return Number(v + o.v);
    }
    Number operator-(Number o) const {
        if (joined == 1 && o.product) return Number(std::fmaf(-o.a, o.b, v));
        if (joined == 2 && product) return Number(std::fmaf(a, b, -o.v));
        return Number(v - o.v);
    }
    bool operator>(Number o) const { return v > o.v; }
    bool operator==(Number o) const { return v == o.v; }
};
static Number operator*(float a, Number b) { return Number(a, b.v); }
static Number fmaf(Number a, Number b, Number c) { return Number(std::fmaf(a.v, b.v, c.v)); }
static Number copysignf(Number a, Number b) { return Number(std::copysign(a.v, b.v)); }
static Number __fmul_rn(Number a, Number b) { return Number(a.v * b.v); }
static Number __fsub_rn(Number a, Number b) { return Number(a.v - b.v); }
#define float Number
%s
#undef float
extern "C" float decided(float x, float c, float a, int how) { joined = how; return decided_code(x, c, a).v; }
"""


@pytest.fixture(scope="module")
def decided(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("a compiler for the host is needed")
    with open(HEADER) as handle:
        text = handle.read()
    start = text.index("__device__ __forceinline__ float decided_code(")
    folder = tmp_path_factory.mktemp("rounding")
    (folder / "decided.cpp").write_text(SHIMS % text[start:text.index("\n}\n", start) + 3])
    subprocess.run(["g++", "-O2", "-ffp-contract=off", "-shared", "-fPIC", "-o", str(folder / "decided.so"), str(folder / "decided.cpp")], check=True)
    call = ctypes.CDLL(str(folder / "decided.so")).decided
    call.argtypes, call.restype = [ctypes.c_float] * 3 + [ctypes.c_int], ctypes.c_float
    return call


@pytest.mark.parametrize("joined", [0, 1, 2])
@pytest.mark.parametrize("exponent", [-96, -20, 0, 99, 126])
def test_codes_next_to_the_middle_of_two(decided, exponent, joined):
    rng = np.random.default_rng(exponent + 200)
    checked = 0
    while checked < 2000:
        a = np.ldexp(np.float32(rng.uniform(1, 2)), exponent)
        x = np.float32(float(a) * (rng.integers(-126, 126) + 0.5) / 127)
        for _ in range(int(rng.integers(0, 3))):
            x = np.nextafter(x, np.float32(rng.choice([-np.inf, np.inf])))
        value = 127 * Fraction(float(x)) / Fraction(float(a))
        below = value.numerator // value.denominator
        over = value - below
        want = below + (over > Fraction(1, 2) or (over == Fraction(1, 2) and below % 2))
        for c in (below, below + 1):                 # either neighbour may be the one that the factor's product was rounded to
            assert decided(x, c, a, joined) == want, (x, c, a)
        checked += 1
