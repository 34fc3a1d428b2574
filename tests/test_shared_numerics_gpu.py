"""Numerics of attention over shared positions that its outputs' own rounding would hide: the bits of the weights, and of a
quantized cache's values, that meet in its products."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32, Q4_0, Q8_0
from tests.test_paged_gpu import IDS, IO
from tests.test_shared_steps_gpu import Steps

pytestmark = pytest.mark.gpu

# What a product may be off by, relative. Of two bf16 terms, each rounded, the first leaves 2^-8 at most of a number in [1, 2) and the
# second half of 2^-16: 2^-17; so over a bf16 cache for its rows. Over a quantized one for bf16 rows both factors are off by
# that, and the product of what their first terms leave, 2^-16, is left out: 2^-15. Of two fp16 terms 2^-11 and half of
# 2^-21: 2^-22. Else the terms hold all 24 bits, and what is left out is 2 * 2^-8 * 2^-17.
TERMS = {(BF16, BF16): 2.0**-17, (Q8_0, BF16): 2.0**-15, (Q4_0, BF16): 2.0**-15, (F16, F16): 2.0**-22, (F16, F32): 2.0**-22,
         (F32, F32): 0.0, (BF16, F32): 0.0}


def in_terms(io, x, n=3):
    """n numbers of a type that add up to x."""
    out = []
    for _ in range(n):
        t = float(ref.from_type(io, ref.to_type(io, np.full(1, x, np.float32)))[0])
        out.append(t)
        x -= t
    return out


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [2, 20], ids=["few", "many"])
def test_weights_and_values_keep_their_bits(hip, cache, io, hd, rows):
    """Every other position has a weight of 0.5 + 2^-8 - 2^-21 and values of about 1, of which cut-off bf16 terms would lose the most
    (quantized: values of 1 + 2^-7 - 2^-19 too); those between weigh 1 and have values that nearly cancel them. 64 positions:
    64 additions of 2^-24 each, exp2 2^-22, a score's roundings 2^-21 in all."""
    n, quant = 64, cache in (Q8_0, Q4_0)
    w = 0.5 + 2.0**-8 - 2.0**-21
    k, v, q = np.zeros((n, 1, hd), np.float32), np.empty((n, 1, hd), np.float32), np.zeros((rows, 1, 4, hd), np.float32)
    q[..., :1 if quant else 3] = 1.0
    k[1::2, 0, :1 if quant else 3] = np.log(w) if quant else in_terms(cache, np.log(w))
    v[1::2] = 1 + 2.0**-7 - 2.0**-19 if quant else 1.0
    # (quantized: between two numbers of 16 bits; else one of 8)
    v[::2] = -(np.rint(w * v[1, 0, 0] * 2.0**16) + 0.25) * 2.0**-16 if quant else -(0.5 + 2.0**-8)
    c = Steps(np.random.default_rng(1), cache, io, hd, 1, 4, rows, [4], n, k=k, v=v, q=q, scale=1.0)
    assert (c.lens == n).all()
    raw, _ = c.run()
    got = ref.from_type(io, raw).astype(np.float64)
    assert (got == got[:1, :1]).all()
    out, _, _, mean = ref.attention64(c.q[0, :1], c.k, c.v, 1.0)
    p = np.exp(c.k[1, 0].astype(np.float64) @ c.q[0, 0])
    assert abs(p / w - 1) < 2.0**-22 and (np.abs(out) < 2.0**-15).all()
    tol = (TERMS.get((cache, io), 2.0**-24) + 2.0**-18 + 2.0**-22 + 2.0**-21) * mean + ref.HALF_STEP[io] * np.abs(out) + (2.0**-25 if io == F16 else 0)
    assert (np.abs(got[0, :1] - out) <= tol).all(), (np.abs(got[0, :1] - out) / mean).max() * 2.0**17
