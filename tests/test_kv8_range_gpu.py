"""GPU tests of attention over the paged 8-bit cache where values, keys or
queries take sizes far from a model's: against 64 bits, through the few-row and
the many-row kernel.

Bound, from the kernels' arithmetic (u = 2^-24).  x is a score in powers of two,
w_t = p_t |v_t| what token t gives to an element:
* a score is off by ds <= size (2^-22 + 2 d u) + 2^-22 (size + 256): the first
  part from q's bits and the sums, the second from x - m and log2 of the value
  scale, whose magnitudes stay below 1.45 size + 256, in f32 (half an ulp each,
  and three such operations);
* every weight is off by a factor exp(2 ds), its rounding to f16 (2^-11) or
  hi + lo (2^-21) and the sums' 2^-18; a weight below 2^-32 of the largest
  p_t * scale_t may vanish, and counts up to 127 of its scale;
* the output is rounded to its type."""
import numpy as np
import pytest

from tests.test_kv8_gpu import dt, ids, make, put

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t

    assert _t.cuda.is_available()
    return _t


def check_weighted(torch, c, r, s, n, heads, dtype, q, window=0, sinks=0, floor=0.0):
    """attend's results for the last n tokens of s against 64 bits, each element within what its own terms allow.
    floor: the error of an element of q, of the row's largest."""
    scale = r.d ** -0.5
    out, lse = c.attend(0, q, seqs=ids(torch, [s]), n=n, window=window, sinks=sinks, return_lse=True)
    c.check()
    got, z = out.float().cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    qh = q.float().cpu().numpy().astype(np.float64)
    k, v = r.values(0, s, 0), r.values(0, s, 1)
    length, u = len(k), 2.0 ** -24
    vs = np.zeros((length, r.kv))
    for t in range(length):
        vs[t] = r.scale[1, 0, r.table[s, t // r.page], :, t % r.page // r.block]
    pos = length - n + np.arange(n)
    t = np.arange(length)
    see = t[None] <= pos[:, None]
    if window:
        see &= (t[None] > pos[:, None] - window) | (t[None] < sinks)
    wt, rnd = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11, torch.finfo(q.dtype).eps / 2
    for h in range(heads):
        kh, vh, sh = k[:, h * r.kv // heads], v[:, h * r.kv // heads], vs[:, h * r.kv // heads]
        x = np.where(see, qh[:, h] @ kh.T * scale, -np.inf)
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        p = e / e.sum(1, keepdims=True)
        ref, rl = p @ vh, m[:, 0] + np.log(e.sum(1))
        size = np.where(see, np.abs(qh[:, h]) @ np.abs(kh).T, 0).max(1) * scale
        reach = np.abs(qh[:, h]).max(1) * np.where(see, np.abs(kh).sum(1)[None], 0).max(1) * scale
        ds = floor * reach + size * (2.0 ** -22 + 2 * r.d * u) + 2.0 ** -22 * (size + 256)
        tol = (p @ np.abs(vh)) * (np.exp(2 * ds) - 1 + wt + 2.0 ** -18)[:, None] + \
            length * 2.0 ** -32 * 127 * (p * sh).max(1)[:, None]
        err = np.abs(got[:, h] - ref)
        # half a step of the type, which is fixed below its normal numbers
        fi = torch.finfo(q.dtype)
        limit = tol + np.maximum(rnd * np.abs(ref), fi.tiny * fi.eps / 2)
        bad = ~(err <= limit)
        assert not bad.any(), (h, int(bad.sum()), float(got[:, h][bad][0]), float(ref[bad][0]), float(limit[bad][0]))
        assert np.all(np.abs(z[:, h] - rl) <= ds + 2.0 ** -18 + 2.0 ** -21 * np.abs(rl))


def filled(torch, keys, values, block=16):
    """A cache of one sequence (and a second, empty one) with these rows [n, kv, d], and its model."""
    n, kv, d = keys.shape
    c, r = make(torch, d=d, kv=kv, page=32, block=block, n_seqs=2, max_pages=-(-n // 32), n_pages=-(-n // 32) + 3)
    assert r.reserve([1], [n])
    c.reserve(ids(torch, [n]), seqs=ids(torch, [1]))
    put(torch, c, r, [1], [n], [torch.tensor(x.astype(np.float32), device="cuda") for x in (keys, values)])
    return c, r


def queries(torch, rng, n, heads, d, dtype, size):
    return torch.tensor(rng.standard_normal((n, heads, d)) * size, dtype=torch.float32, device="cuda").to(dt(torch, dtype))


def powers(rng, kind, n):
    """log2 of the values' size in every block of 16 tokens."""
    nb = -(-n // 16)
    e = {"huge": lambda: np.full(nb, 127.9), "to huge": lambda: rng.uniform(60, 127.9, nb),
         "tiny": lambda: np.full(nb, -99.0), "to tiny": lambda: rng.uniform(-99, -40, nb),
         # ordinary values, and a few blocks of huge ones
         "some huge": lambda: np.where(rng.random(nb) < 0.1, rng.uniform(85, 127.9, nb), rng.uniform(-12, 12, nb)),
         "huge late": lambda: np.where(np.arange(nb) == nb - 2, 127.9, rng.uniform(-12, 12, nb)),
         "huge first": lambda: np.where(np.arange(nb) == 0, 127.9, rng.uniform(-12, 12, nb)),
         "tiny and ordinary": lambda: np.where(rng.random(nb) < 0.5, rng.uniform(-99, -60, nb), 0.0)}[kind]()
    return e.repeat(16)[:n]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 60])
@pytest.mark.parametrize("kind", ["huge", "to huge", "tiny", "to tiny", "some huge", "huge late", "huge first",
                                  "tiny and ordinary"])
def test_values_of_any_size(torch, kind, rows, dtype):
    """From the smallest a scale holds to the largest finite one; few and many rows (4 heads on one), pasts of
    one item and of several parts, even scores and scores that leave nearly all weight to one token."""
    rng = np.random.default_rng(len(kind) * 7 + rows)
    for n, d in ((300, 128), (3000, 64)):
        e = powers(rng, kind, n)
        x = rng.uniform(-1, 1, (n, 1, d))
        c, r = filled(torch, rng.standard_normal((n, 1, d)), x * np.exp2(e)[:, None, None])
        for size in (0.3, 1.5, 12.0):
            check_weighted(torch, c, r, 1, rows, 4, dtype, queries(torch, rng, rows, 4, d, dtype, size))
        check_weighted(torch, c, r, 1, rows, 4, dtype, queries(torch, rng, rows, 4, d, dtype, 1.5), window=n // 3, sinks=5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 60])
def test_huge_values_that_a_row_hardly_sees(torch, rows, dtype):
    """One block of 2^120 whose scores lie 60 to 110 powers of two below the others': its values count, and the
    ordinary ones' weights keep their bits."""
    rng = np.random.default_rng(rows)
    n, d = 700, 64
    for below in (60.0, 90.0, 110.0, 119.0):
        keys = np.zeros((n, 1, d))
        keys[:, 0, 0] = 1.0
        keys[:, 0, 1] = rng.standard_normal(n) * 0.02
        at = slice(208, 224)
        keys[at, 0, 0] = -1.0
        e = np.zeros(n)
        e[at] = 120.0
        c, r = filled(torch, keys, rng.uniform(-1, 1, (n, 1, d)) * np.exp2(e)[:, None, None])
        q = np.zeros((rows, 4, d))
        q[..., 0] = below * np.log(2.0) / 2 * d ** 0.5
        q[..., 1] = rng.standard_normal((rows, 4))
        check_weighted(torch, c, r, 1, rows, 4, dtype, torch.tensor(q, dtype=torch.float32, device="cuda").to(dt(torch, dtype)))


@pytest.mark.parametrize("rows", [1, 60])
def test_tiny_values_of_a_long_past(torch, rows):
    """40000 tokens of values near 1e-30: the sum of their weights stays finite."""
    rng = np.random.default_rng(rows)
    n, d = 40000, 64
    c, r = filled(torch, rng.standard_normal((n, 1, d)), rng.uniform(-1, 1, (n, 1, d)) * 2.0 ** -99, block=32)
    check_weighted(torch, c, r, 1, rows, 4, "f32", queries(torch, rng, rows, 4, d, "f32", 0.3))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 60])
def test_growing_keys_and_scales_far_apart(torch, rows, dtype):
    """Scores that grow along the past (the references move in every tile) over value blocks between 2^-20 and 2^12,
    for small, ordinary and large queries."""
    rng = np.random.default_rng(rows)
    n, d = 700, 128
    x = rng.standard_normal((n, 1, d))
    grow = np.linspace(0.01, 4, n)[:, None, None]
    e = rng.integers(-20, 10, -(-n // 16)).repeat(16)[:n]
    c, r = filled(torch, x * grow, x * np.exp2(e)[:, None, None])
    for size in (1e-4, 1.0, 20.0):
        check_weighted(torch, c, r, 1, rows, 4, dtype, queries(torch, rng, rows, 4, d, dtype, size))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [300, 2500])
def test_rows_that_are_not_finite_spoil_themselves_only(torch, n, dtype):
    """In the many-row kernel, whole items and split ones."""
    rng = np.random.default_rng(n)
    rows, d = 60, 64
    c, r = filled(torch, rng.standard_normal((n, 1, d)), rng.standard_normal((n, 1, d)))
    q = queries(torch, rng, rows, 4, d, dtype, 1.5)
    clean, lse = c.attend(0, q, seqs=ids(torch, [1]), n=rows, return_lse=True)
    bad = [(0, 0, float("nan")), (31, 2, float("inf")), (32, 0, -float("inf")), (59, 3, float("nan"))]
    q2, keep = q.clone(), torch.ones(rows, 4, dtype=torch.bool)
    for t, h, x in bad:
        q2[t, h, (t * 7) % d] = x
        keep[t, h] = False
    got, lse2 = c.attend(0, q2, seqs=ids(torch, [1]), n=rows, return_lse=True)
    assert torch.isnan(got[~keep]).all() and not torch.isfinite(lse2[~keep]).any()
    assert torch.equal(got[keep], clean[keep]) and torch.equal(lse2[keep], lse[keep])
    c.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 60])
def test_queries_of_many_sizes_in_one_row(torch, rows, dtype):
    """A row is held relative to its largest element: each element is off by at most 2^-38 of that.  Rows with an
    element near 60000 that no key has any of, beside subnormal f16 numbers and ordinary ones that decide."""
    rng = np.random.default_rng(rows)
    n, d = 300, 64
    keys = rng.standard_normal((n, 1, d)) * 3000.0
    keys[..., :2] = 0.0
    c, r = filled(torch, keys, rng.standard_normal((n, 1, d)))
    q = np.exp2(rng.uniform(-24, -10, (rows, 4, d))) * rng.choice([-1, 1], (rows, 4, d))
    q[..., 0] = rng.uniform(30000, 65000, (rows, 4))
    q[: rows // 2, :, 0] = 2.0  # some rows without it
    q = torch.tensor(q, dtype=torch.float32, device="cuda").to(dt(torch, dtype))
    check_weighted(torch, c, r, 1, rows, 4, dtype, q, floor=2.0 ** -38)
