"""ops.PagedCache with more sequences than a prefill call takes, against numpy in 64
bits."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import HD, bits, expect, filled, packed, rng_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("B", [128, 129, 300])
def test_prefill_of_any_batch(B, dtype):
    rng = rng_of("any batch", B)
    H, hkv, page = 6, 2, 32
    new = [int(x) for x in rng.integers(0, 30, B)]
    past = [int(x) for x in rng.integers(0, 90, B)]
    new[-1], past[-1] = 7, 400
    lens = [a + b for a, b in zip(new, past)]
    c, K, V = filled(rng, lens, hkv, page)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    n, f16 = int(cu[-1]), dtype == np.float16
    q = rng.standard_normal((n + 9, H * HD)).astype(dtype)
    before = rng.standard_normal(q.shape).astype(dtype)
    got = c.attn_prefill(q, cu, before)
    assert np.array_equal(bits(got[n:]), bits(before[n:]))
    for z, m in enumerate(new):
        at = slice(cu[z], cu[z + 1])
        want, tol = expect(q[at], K[z], V[z], hkv, lens[z] - m, f16, 1 if f16 else 2)
        ref.check_rows(got[at], want, tol, z)
