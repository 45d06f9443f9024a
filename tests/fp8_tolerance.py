"""How far the 8-bit attention kernels may be from float64, from their arithmetic.

A score is an fp32 sum of D exact products (three times as many for an fp32 query, whose parts add up
to it); each of its additions is off by at most 2^-23 of the terms' absolute sum A (a rounding, or a
truncation inside the matrix core), the two multiplications by scales and log2 e by 2^-24 each and the
subtraction of the maximum by 2^-24 of the score.  So the exponent's error, in units of ln, is at most
(D + 8) 2^-23 A.  A weight then carries that, the exponential's own error and the parts it is split
into: 2^-17 for two bf16 parts, 2^-25 for three.  Sums over the tokens add 2^-23 per addition of a
wave's partial sum, at most n of them.  Numerator and denominator both carry it: twice the whole, times
the largest |v|.  Last the rounding of the output, half a step.
"""

import numpy as np

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def attention_bound(want, bound, vmax, n, d, dtype, out_dtype):
    """Largest allowed |got - want|, the shape of want [.., Hq, D]; bound [.., Hq]: A; n: tokens."""
    terms = 3 * d if dtype == "float32" else d
    parts = 2.0 ** -25 if dtype == "float32" else 2.0 ** -17
    rel = (terms + 8) * 2.0 ** -23 * bound[..., None] + 2.0 ** -22 + parts + n * 2.0 ** -23
    return 2 * vmax * rel + HALF_STEP[out_dtype] * (np.abs(want) + 2 * vmax * rel) + 2.0 ** -25   # fp16's least step / 2
