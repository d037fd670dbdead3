"""Taking rows of the newest block back on the GPU: also where the last append has
completed the block."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import FMTS, HD, bits, held, new_cache, rng_of, rows, set_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sizes", [[64], [40, 24], [63, 1], [1] * 64, [31, 33], [32, 32], [5, 27, 32]])
@pytest.mark.parametrize("back", [63, 60, 33])
def test_rewind_from_a_completed_block(fmt, sizes, back):
    """64 rows by appends of any sizes, then others from `back` on: within the block that
    the last of them completed, past its end too."""
    rng = rng_of("rewind64", fmt, sizes, back)
    k, v = rows(rng, 2, 2, 64)
    k[:, :, 63, 5] *= 40                                    # its scale goes with it
    k2, v2 = rows(rng, 2, 2, 40)
    c = new_cache(2, 2, 160, fmt)
    at = 0
    for s in sizes:
        c.append(k[:, :, at:at + s], v[:, :, at:at + s], [at, at])
        at += s
    m = [3, 40]                                             # within the block, and past it
    c.append(k2, v2, [back, back], m)
    gk, gv = c.read([0, 0], 104)
    for z in range(2):
        n = back + m[z]
        for got, x, y in ((gk, k, k2), (gv, v, v2)):
            want = held(np.concatenate([x[z, :, :back], y[z, :, :m[z]]], 1), n, fmt)
            assert np.array_equal(bits(got[z, :, :n]), bits(want)), z


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("inplace", [True, False])
def test_rewind_after_a_cut(fmt, inplace):
    """A cut of whole blocks keeps the newest block's rows for it."""
    rng = rng_of("rewind cut", fmt, inplace)
    k, v = rows(rng, 1, 1, 192)
    k2, v2 = rows(rng, 1, 1, 9)
    c = new_cache(1, 1, 192, fmt)
    c.append(k, v, [0])
    w = rng.random((1, 1, 6)).astype(np.float32)
    set_weights(c, w)
    d = c if inplace else new_cache(1, 1, 96, fmt)
    new = c.evict([192], 3, 1, 1, None if inplace else d)
    assert new.tolist() == [96]
    keep = ref.kept_blocks(w[0, 0], 6, 3, 1, 1)
    at = np.concatenate([np.arange(32 * b, 32 * b + 32) for b in keep])[:85]
    d.append(k2, v2, [85])
    gk, gv = d.read([0], 94)
    for got, x, y in ((gk, k, k2), (gv, v, v2)):
        want = held(np.concatenate([x[0][:, at], y[0]], 1), 94, fmt)
        assert np.array_equal(bits(got[0]), bits(want))


def test_rewind_leaves_other_rows_of_the_cache():
    """The rows kept for it are the head's own: nothing else of the cache changes when
    an append completes a block."""
    c = new_cache(2, 2, 64, 0)
    k, v = rows(rng_of("tail"), 2, 2, 32)
    before = c.data.download()
    c.append(k, v, [0, 0], [32, 0])
    after = c.data.download()
    assert np.array_equal(after[1], before[1])
    al = lambda b: (b + 255) // 256 * 256  # noqa: E731
    tails = al(2 * 2 * 8192) + al(2 * 2 * 8) + al(2 * 2 * 4)
    kept = after[0, tails:tails + 2 * 2 * 32 * HD * 2].view(np.float16).reshape(2, 2, 32, HD)
    assert np.array_equal(kept[:, 0].view(np.uint16), k[0].view(np.uint16))
    assert np.array_equal(kept[:, 1].view(np.uint16), v[0].view(np.uint16))
    for h in range(2):                                      # the second block of each head is not begun
        at = (2 * h + 1) * 8192
        assert np.array_equal(after[0, at:at + 8192], before[0, at:at + 8192])
