"""GPU tests of the paged 8-bit cache with thousands of sequences in a call,
single tokens and prompt chunks among one another."""
import numpy as np
import pytest

from tests.test_kv8_gpu import check_attend, fill, make, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t

    assert _t.cuda.is_available()
    return _t


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_thousands_of_sequences(torch, dtype):
    rng = np.random.default_rng(1)
    m = 3000
    c, r = make(torch, d=64, kv=1, page=16, block=16, n_seqs=m, max_pages=8, n_pages=4 * m)
    order = [int(x) for x in rng.permutation(m)]
    fill(torch, c, r, order, [int(x) for x in rng.integers(0, 40, m)], rng, dtype)
    fill(torch, c, r, order, [1] * m, rng, dtype)
    check_attend(torch, c, r, order, [1] * m, 2, dtype, rng)
    # a few chunks among single tokens, some sequences without rows
    counts = [int(x) for x in rng.choice([0, 1, 1, 1, 1, 2], m)]
    for i in rng.integers(0, m, 20):
        counts[i] = int(rng.integers(20, 50))
    fill(torch, c, r, order, counts, rng, dtype)
    check_attend(torch, c, r, order, counts, 2, dtype, rng)
    check_attend(torch, c, r, order, counts, 2, dtype, rng, window=20, sinks=3)
    k, v = c.rows(0, n=2)
    for s in (0, 17, m - 1):
        want = [np.concatenate([np.zeros((2, 1, 64)), r.values(0, s, z)])[-2:] for z in range(2)]
        assert np.array_equal(k[2 * s:2 * s + 2].cpu().numpy(), want[0].astype(np.float32))
        assert np.array_equal(v[2 * s:2 * s + 2].cpu().numpy(), want[1].astype(np.float32))
    c.check()
    same(torch, c, r)
