"""The 2^t that draft verification sums its weights with (verify.hip): the same coefficients and operations in IEEE double
arithmetic, against 2^t to 50 digits."""
import os
import re
from decimal import Decimal, getcontext
from fractions import Fraction

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a100-vision-infer_amd", "csrc", "verify.hip")


def worst(degree):
    """The largest relative error of the polynomial of that degree over [-1/2, 1/2], every operation rounded once."""
    getcontext().prec = 50
    ln2 = 0.693147180559945309417
    c, v = [], 1.0
    for k in range(degree + 1):
        c.append(v)
        v *= ln2 / (k + 1)
    top = Decimal(0)
    for i in range(-2000, 2001):
        f = i / 4000
        p = c[-1]
        for k in range(degree - 1, -1, -1):
            p = float(Fraction(p) * Fraction(f) + Fraction(c[k]))  # a fused multiply-add: rounded once
        top = max(top, abs(Decimal(p) / Decimal(2) ** Decimal(f) - 1))
    return float(top)


def test_error_of_the_polynomial():
    text = open(SOURCE).read()
    degree = int(re.search(r"double c\[(\d+)\]", text).group(1)) - 1
    stated = float(re.search(r"relative error of at most (\d+e-\d+)", text.replace("\n// ", " ")).group(1))
    got = worst(degree)
    assert 0.5 * stated < got <= stated, (got, stated)
