"""Precision of the attention's weights: where the values cancel, what the weights lose to a rounding shows in full."""
import numpy as np
import pytest

from conftest import bf16_bits, bf16_vals
from serving_kit import BF16_HALF_STEP, F32_HALF_STEP, Device, attention64
from test_gpu_serving_attention import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (14, 2, 64), (40, 2, 128), (64, 1, 64)])
@pytest.mark.parametrize("c", [0.296875, 1.1015625, 2.703125])
def test_weights_are_not_rounded_to_bf16(tiny_model, heads, kv, dim, c):
    """Every 16th key has the weight 1, the others exp(-c), no power of two, and the same values, which the 16th ones' take away again.  All
    weights but those of 1 lose the same share to a rounding, so an error of the weights is an error of half that share of sum p |v|.

    Allowed: the result's own rounding; the weights' as a sum of two bf16 numbers, a half step of a half step; the scores' errors in
    numerator and denominator; fp32 sums, of two terms per key in the numerator and one in the denominator.  A weight that is
    rounded to bf16 once is off by 2^-9 to 2^-11 here, half of that in the result, against 2^-12 allowed."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(96, [(40, 1), (40, 2), (40, 3)]), (96, [(40, 1)])], heads, kv, dim, 16, seed=int(8 * c))
        n, book = 136, s.c.book
        ones = -(-n // 16)
        u = bf16_vals(bf16_bits(s.rng.standard_normal(dim)))
        book.k[..., 3] = bf16_bits(np.array([-c]))[0]
        book.v[:] = bf16_bits(u)
        book.k[..., 0, 3] = 0
        book.v[..., 0, :] = bf16_bits(-(n - ones) / ones * np.exp(-c) * u)
        dev.put(book.k, s.c.at["k"])
        dev.put(book.v, s.c.at["v"])
        s.q[:] = 0
        s.q.reshape(-1, heads, dim)[:, :, 3] = bf16_bits(np.array([1.0]))[0]
        for b in (s.batch(), s.batch(max_len=1040), s.batch(grouped=False, max_len=1040)):
            out, _ = s.run(b, scale=1.0)
            for i, q in enumerate(s.seqs):
                rows = slice(s.cu[i], s.cu[i + 1])
                x = bf16_vals(s.q[rows]).astype(np.float64).reshape(-1, heads, dim)
                k, v = book.keys(s.layer, q)
                want, _, size, slack = attention64(x, k, v, n, len(x), heads, 1.0)
                got = bf16_vals(out[rows]).astype(np.float64).reshape(want.shape)
                allowed = BF16_HALF_STEP ** 2 + 2 * slack[..., None] + 3 * (n + 64) * F32_HALF_STEP
                tol = BF16_HALF_STEP * np.abs(want) * (1 + 1e-3) + allowed * size + 1e-30
                assert (np.abs(got - want) <= tol).all(), (i, (np.abs(got - want) / tol).max())
