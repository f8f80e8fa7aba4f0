"""The polynomial that stands for a part of exp2 in attention over the 8-bit cache, evaluated as the kernel does: in
float32, Horner's scheme with one rounding per multiply-add."""
import pathlib
import re

import numpy as np

SOURCE = pathlib.Path(__file__).resolve().parent.parent / "bladedisc_b200" / "csrc" / "kernels" / "kv8_prefill.cu"


def coefficients():
    text = SOURCE.read_text()
    body = text[text.index("uint64_t exp2_pair("):]
    body = body[:body.index("\n}\n")]
    c = [np.float32(m) for m in re.findall(r"pair\(([0-9.e+-]+)f, \1f\)", body)]
    return [x for x in c if x not in (np.float32(12582912), np.float32(-12582912), np.float32(-1))]


def exp2(x):
    """2^x for float32 x as the kernel computes it, in float64 with a rounding to float32 after every operation."""
    x = np.maximum(x, np.float32(-125))
    r = x + np.float32(12582912)
    f = x - (r - np.float32(12582912))  # exact
    c = coefficients()
    y = np.full_like(x, c[0])
    for k in c[1:]:
        y = (y.astype(np.float64) * f + np.float64(k)).astype(np.float32)
    n = (r - np.float32(12582912)).astype(np.int32)
    return np.ldexp(y, n)


def test_relative_error():
    assert len(coefficients()) == 6
    # every float32 of [1/4, 1/2] and the like is too many: a fine grid, and the places where n changes
    x = np.concatenate([np.linspace(-60, 13, 2_000_003), np.arange(-60, 13) + 0.5, np.nextafter(np.arange(-60, 13) + 0.5, 99),
                        np.arange(-60, 14)]).astype(np.float32)
    err = np.abs(exp2(x).astype(np.float64) / np.exp2(x.astype(np.float64)) - 1)
    # the polynomial's own error, 2^-22.62; the last rounding, 2^-24 of values from 1 on; the one before, 2^-25 times
    # |f| <= 1/2; those before that, a quarter of it in all: (1.55 + 0.60 + 0.15 + 0.04) 10^-7 < 2^-22
    assert err.max() < 2.0 ** -22
    assert exp2(np.float32([-125, -1e30, 0])).tolist() == [2.0 ** -125 * exp2(np.float32([0]))[0]] * 2 + [exp2(np.float32([0]))[0]]
