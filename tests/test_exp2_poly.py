"""The FMA-pipe exponential of the paged tcgen05 attention, evaluated on the CPU
as the kernel does (fp32, one rounding a step), against 2^x in 64 bits."""
import os
import re

import numpy as np

import hackthenorth_b200

SOURCE = os.path.join(os.path.dirname(hackthenorth_b200.__file__), "csrc", "paged_attention_tc.cuh")


def test_polynomial_is_as_exact_as_its_comment_says():
    text = open(SOURCE).read()
    coefficients = [np.float32(1)] + [np.float32(re.search(rf"kC{i} = ([0-9.]+)f", text).group(1)) for i in range(1, 6)]
    f32 = lambda x: x.astype(np.float32)
    x = f32(np.concatenate((np.linspace(-127, 8, 2000001), np.arange(-127, 9))))
    bias = np.float32(12582912.0 + 127.0)  # as kRound
    n = f32(x + bias)
    f = f32(x + f32(bias - n))
    p = np.full_like(x, coefficients[5])
    for c in coefficients[4::-1]:
        p = f32(p.astype(np.float64) * f + c)
    scale = (n.view(np.uint32) << np.uint32(23)).view(np.float32)
    got = f32(p * scale).astype(np.float64)
    normal = x >= -125
    error = np.abs(got / np.exp2(x.astype(np.float64)) - 1)[normal]
    assert error.max() <= 2.0 ** -22.4
    assert got[x == -127].max() == 0.0 and bool((got >= 0).all())
    whole = normal & (x == np.rint(x))
    assert whole.sum() > 100 and np.array_equal(got[whole], np.exp2(x[whole].astype(np.float64)))
