"""GPU tests of what the paged 8-bit cache does with batches that are wrong in
ways only the device can see: it says so in the status word, and nothing
outside the batch changes."""
import numpy as np
import pytest

from tests.test_kv8_gpu import fill, ids, make, put, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t

    assert _t.cuda.is_available()
    return _t


def fails(torch, c, text):
    from stealcode_b200._lib import SC_ERR_INVALID, ScError

    with pytest.raises(ScError, match=text) as e:
        c.check()
    assert e.value.code == SC_ERR_INVALID
    c.clear_status()


BAD_CU = [("more rows than n", [0, 5, 8], 3, 8), ("fewer than none", [0, 6, 4], 6, 8), ("before the rows", [-2, 3, 5], 5, 8),
          ("past the rows", [0, 3, 11], 8, 8), ("far past the rows", [0, 2, 2 ** 31 - 1], 2 ** 20, 8),
          ("more rows than a long n", [0, 70, 90], 40, 90), ("long, fewer than none", [0, 60, 41], 60, 60),
          ("long, before the rows", [-(2 ** 31), 45, 60], 60, 60)]


@pytest.mark.parametrize("what,cu,n,total", BAD_CU, ids=[x[0] for x in BAD_CU])
def test_rows_that_cu_does_not_describe(torch, what, cu, n, total):
    rng = np.random.default_rng(n % 1000)
    c, r = make(torch, d=64, kv=2, page=16, block=16, n_seqs=4, max_pages=10, n_pages=40)
    fill(torch, c, r, [0, 1, 2], [100, 120, 60], rng)
    seqs = ids(torch, [1, 0])
    bad = [not (0 <= a <= b <= total and b - a <= n) for a, b in zip(cu, cu[1:])]
    q = torch.tensor(rng.standard_normal((total, 4, 64)), dtype=torch.float32, device="cuda")
    out = torch.full_like(q, 7.0)
    c.attend(0, q, seqs=seqs, cu=ids(torch, cu), n=n, out=out)
    fails(torch, c, "cu")
    covered = torch.zeros(total, dtype=torch.bool)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):  # entries that are right have their results
        if not bad[i]:
            covered[a:b] = True
            want = c.attend(0, q[a:b].contiguous(), seqs=seqs[i:i + 1], n=b - a) if b > a else q[:0]
            assert torch.allclose(out[a:b], want, atol=1e-5, rtol=0)
    assert any(bad) and (out[~covered] == 7.0).all()  # the others' rows are not touched
    c.rows(0, seqs=seqs, cu=ids(torch, cu), n=n, total=total)
    fails(torch, c, "cu")
    x = torch.ones(total, 2, 64, device="cuda")
    keep = c.k.clone(), c.k_scale.clone(), c.v.clone(), c.v_scale.clone()
    c.append(0, x, x, seqs=seqs, cu=ids(torch, cu), n=n)
    fails(torch, c, "cu")
    for s in [2] + [s for s, b in zip((1, 0), bad) if b]:
        for t, old in zip((c.k, c.k_scale, c.v, c.v_scale), keep):
            pages = c.table[s][c.table[s] >= 0].long()
            a, b = t[:, pages].nan_to_num(3.0), old[:, pages].nan_to_num(3.0)
            assert torch.equal(a, b), s


def test_packed_rows_of_no_entry_are_not_touched(torch):
    """Packed rows before the first entry and after the last, as buffers of a fixed size have: no failure."""
    rng = np.random.default_rng(3)
    c, r = make(torch, d=64, kv=2, page=16, block=16, n_seqs=3, max_pages=10)
    fill(torch, c, r, [0, 1], [50, 80], rng)
    for cu, n, total in (([4, 5, 6], 1, 9), ([3, 40, 60], 40, 64)):
        q = torch.tensor(rng.standard_normal((total, 4, 64)), dtype=torch.float32, device="cuda")
        out = torch.full_like(q, 7.0)
        c.attend(0, q, cu=ids(torch, cu), n=n, out=out)
        c.check()
        assert (out[:cu[0]] == 7.0).all() and (out[cu[-1]:] == 7.0).all() and (out[cu[0]:cu[-1]] != 7.0).all()
    x = [torch.tensor(rng.standard_normal((64, 2, 64)), dtype=torch.float32, device="cuda") for _ in range(2)]
    assert r.reserve([0, 1], [37, 20])
    c.reserve(ids(torch, [37, 20]))
    c.append(0, *x, cu=ids(torch, [3, 40, 60]), n=37)
    h = [y.cpu().numpy() for y in x]
    r.append(0, [0, 1], [h[0][3:40], h[0][40:60]], [h[1][3:40], h[1][40:60]])
    c.check()
    same(torch, c, r)


@pytest.mark.parametrize("n", [1, 60])
def test_attend_reports_sequences_outside_the_cache(torch, n):
    rng = np.random.default_rng(12)
    c, r = make(torch, d=64, kv=1, max_pages=12)
    fill(torch, c, r, [0], [70], rng)
    q = torch.tensor(rng.standard_normal((3 * n, 2, 64)), dtype=torch.float32, device="cuda")
    for seqs in ([7, 0, -1], [0, 1, 4]):
        out, lse = c.attend(0, q, seqs=ids(torch, seqs), n=n, return_lse=True)
        for i, s in enumerate(seqs):
            a = slice(i * n, (i + 1) * n)
            assert bool(out[a].any()) == (s == 0) and bool(torch.isneginf(lse[a]).all()) == (s != 0)
        fails(torch, c, "sequence id")
    # an entry without rows names nothing
    c.attend(0, q[:1], seqs=ids(torch, [0, 99]), cu=ids(torch, [0, 1, 1]), n=1)
    c.check()


@pytest.mark.parametrize("n", [3, 40])
def test_an_append_that_fails_is_repeated(torch, n):
    """One sequence of the batch has no pages for its rows: the call fails, leaves every other sequence alone, and
    the same rows appended again once there are pages give what an append without the failure gives."""
    rng = np.random.default_rng(n)
    c, r = make(torch, d=64, kv=2, page=16, block=16, n_seqs=5, max_pages=10, n_pages=50)
    fill(torch, c, r, [0, 1, 2, 3], [21, 5, 50, 9], rng)
    assert r.reserve([0, 3], [n, n])
    c.reserve(ids(torch, [n, n]), seqs=ids(torch, [0, 3]))
    x = [torch.tensor(rng.standard_normal((3 * n, 2, 64)) * 3, dtype=torch.float32, device="cuda") for _ in range(2)]
    h = [y.cpu().numpy() for y in x]
    keep = c.k.clone(), c.k_scale.clone(), c.v.clone(), c.v_scale.clone()
    c.length[1] += 16 * 8  # tokens that no page was reserved for
    c.append(0, *x, seqs=ids(torch, [0, 1, 3]), n=n)
    fails(torch, c, "page id")
    pages = c.table[2][c.table[2] >= 0].long()
    for t, old in zip((c.k, c.k_scale, c.v, c.v_scale), keep):
        assert torch.equal(t[:, pages].nan_to_num(3.0), old[:, pages].nan_to_num(3.0))
    c.length[1] = 5
    assert r.reserve([1], [n])
    c.reserve(ids(torch, [n]), seqs=ids(torch, [1]))
    c.append(0, *x, seqs=ids(torch, [0, 1, 3]), n=n)
    r.append(0, [0, 1, 3], *[[y[i * n:(i + 1) * n] for i in range(3)] for y in h])
    c.check()
    same(torch, c, r)
