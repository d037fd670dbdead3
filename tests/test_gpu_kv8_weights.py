"""Block weights of the 8-bit cache's attention where the exact ones are known."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import FMTS, HD, new_cache, rng_of

pytestmark = pytest.mark.gpu


def even(n, pos0, G, nb):
    """Each block's weight when every key is 0: query i gives each of its pos0 + i + 1
    positions an equal share."""
    w = np.zeros(nb)
    for i in range(n):
        m = pos0 + i + 1
        seen = np.clip(m - 32 * np.arange(nb), 0, 32)
        w += G * seen / m
    return w


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,pos0,G", [(1, 0, 1), (1, 30, 1), (1, 4998, 1), (1, 9999, 1), (1, 20010, 1), (1, 40002, 4),
                                      (1, 70000, 1), (3, 2999, 2), (40, 700, 4), (130, 3000, 1), (333, 1000, 4)])
def test_prefill_weights_of_even_rows(fmt, n, pos0, G):
    """Keys of 0: p' is a power of two and a row's sums are whole multiples of it, so
    they are exact, and their reference is the same in every block.  Left are a row's
    reciprocal and one product (u each), and the sum over rows of terms above 0: 256
    threads' ceil(rows / 256) of them, 6 steps over lanes, 2 over waves and the block's
    own weight, u each."""
    rng = rng_of("even", fmt, n, pos0)
    total = pos0 + n
    c = new_cache(1, 1, total, fmt)
    c.append(np.zeros((1, 1, total, HD), np.float16),
             rng.standard_normal((1, 1, total, HD)).astype(np.float16), [0])
    q = rng.standard_normal((n, G * HD)).astype(np.float32)
    c.attn_prefill(q, pos0, add_weights=True)
    nb = (total + 31) // 32
    want = even(n, pos0, G, nb)
    rows = n * G
    adds = (rows + 255) // 256 + 9 if rows > 1 else 0
    ref.check_rows(c.weights()[0, 0, :nb], want, (2 + adds) * ref.U * want, (n, pos0))


def test_prefill_weights_of_more_tiles_than_a_plan_orders():
    """525 row tiles in one launch with weights: keys of 0, as above."""
    n, G = 4200, 16
    c = new_cache(1, 1, n, 0)
    c.append(np.zeros((1, 1, n, HD), np.float16), np.ones((1, 1, n, HD), np.float16), [0])
    out = c.attn_prefill(rng_of("tiles").standard_normal((n, G * HD)).astype(np.float32), 0, add_weights=True)
    want = even(n, 0, G, (n + 31) // 32)
    ref.check_rows(c.weights()[0, 0], want, (2 + (n * G + 255) // 256 + 9) * ref.U * want)
    # values of 1: 127 times the f32 nearest 1 / 127, within 2 u of it; attend()'s bound at S = 0
    ref.check_rows(out, np.ones(out.shape), np.full(out.shape, (2 + 16 + n / 32 + 64 + 4) * ref.U))
