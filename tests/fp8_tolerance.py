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


def rounded_weights_bound(want, bound, dev, vmax, n, d, dtype, out_dtype):
    """The same where each weight is rounded to ``dtype`` (u = half a step of it) and the row sum is that of
    the rounded weights: out = sum p (1 + e_j) v / sum p (1 + e_j) with |e_j| <= u is off by at most
    2 u sum_j p_j |v_j - out| = 2 u dev (to first order; u^2 and an fp16 weight below its normal numbers,
    2^-25 of one each, are covered by the margin of 1.05 and the n 2^-25 term).  Rescaled partial sums of
    split keys are fp32."""
    u = HALF_STEP[dtype]
    rel = (d + 8) * 2.0 ** -23 * bound[..., None] + 2.0 ** -22 + n * 2.0 ** -23
    off = 2.1 * u * dev + 2 * vmax * rel + (n * 2.0 ** -24 * vmax if dtype == "float16" else 0.0)
    return off + HALF_STEP[out_dtype] * (np.abs(want) + off) + 2.0 ** -25
