"""Where the arithmetic of the operators around the 4-bit cache has its limits, restated from the constants in the kernels' source.  No GPU."""
import re
import struct
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parents[1] / "prima.cpp_b200" / "csrc"


def test_weights_of_verification_stay_within_the_exponents():
    """2^(y / 16) over all that the floor lets through: positive, within 2^-46, and at the floor so small that a whole row of it counts as nothing."""
    src = (CSRC / "verify.cu").read_text()
    floor, nothing = float(re.search(r"FLOOR = (\S+?);", src)[1]), float(re.search(r"NOTHING = (\S+?),", src)[1])
    assert struct.pack(">d", floor) == struct.pack(">II", int(re.search(r"FLOOR_HIGH = (0x[0-9a-f]+)u", src)[1], 16), 0)
    body = src[src.index("double power_of_two"):src.index("The weights of a row's logits")]
    poly = [float(re.search(r"double p = (\S+);", body)[1])] + [float(x) for x in re.findall(r"fma\(p, r, (\S+?)\)", body)]
    assert len(poly) == 6

    def power(y):
        k = np.rint(y).astype(np.int64)
        r, p = y - k, poly[0]
        for a in poly[1:]:
            p = p * r + a
        bits = (p * 2.0 ** ((k & 15) / 16)).view(np.int64) + ((k >> 4) << 52)      # the exponent's field, by addition
        return bits.view(np.float64)

    y = np.concatenate((np.linspace(floor, 0.0, 400001), -np.geomspace(1e-300, 16.0, 10001), [-0.0, floor]))
    got, want = power(y), 2.0 ** (y / 16)
    assert np.all(got > 0) and np.max(np.abs(got / want - 1)) < 2.0 ** -46
    assert got[-1] * 2.0 ** 30 < nothing < 2.0 ** -960
