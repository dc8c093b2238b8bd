"""GPU tests of the paged 8-bit key/value cache against the plain model in
kv8_ref: codes, scales, tables and counts bit for bit, attention against 64
bits.

Bounds of the attention tests, from the kernels' arithmetic (u = 2^-24):
* a score is a sum of d products of exact codes with a row of q held to 2^-22
  (f32; f16 and bf16 rows are exact), summed in f32 (d u, doubled for sums that
  truncate), then two f32 products and a difference: |ds| <= size (2^-22 + 2 d u)
  + 2^-21 (size + 8), size = scale * max_t sum_d |q_d k_td|;
* a weight is off by a factor exp(2 ds) against the others, and rounded to f16
  (2^-11) or hi + lo (2^-21); sums over the tokens add 2^-18 (f32, up to 2^13
  terms in partial sums); a weight below 2^-32 of the largest may vanish;
* the output is rounded to its type: half its eps of the value (2^-8 bf16,
  2^-11 f16, 2^-24 f32)."""
import numpy as np
import pytest

from tests.kv8_ref import RefCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t

    assert _t.cuda.is_available()
    return _t


def dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def make(torch, n_layers=1, n_pages=40, kv=2, d=64, n_seqs=4, max_pages=8, page=32, block=16, seed=0):
    """A cache whose unused memory holds garbage (NaN scales among it) and its model."""
    from stealcode_b200 import KvCache8

    c = KvCache8(n_layers, n_pages, kv, d, n_seqs, max_pages, page=page, block=block)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-128, 128, t.shape, generator=g, device="cuda"))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda") * 1e20)
        t[torch.rand(t.shape, generator=g, device="cuda") < 0.3] = float("nan")
    return c, RefCache(n_layers, n_pages, kv, d, n_seqs, max_pages, page, block)


def ids(torch, x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def fill(torch, c, r, seqs, counts, rng, dtype="f32", size=1.0, layer=0):
    """Reserve counts[i] tokens of seqs[i] and append random rows, in both."""
    assert r.reserve(seqs, counts)
    c.reserve(ids(torch, counts), seqs=ids(torch, seqs))
    rows = []
    for z in range(2):
        x = rng.standard_normal((sum(counts), r.kv, r.d)) * size
        x *= np.exp(rng.standard_normal((sum(counts), r.kv, 1)) * 0.5)
        rows.append(torch.tensor(x, dtype=torch.float32, device="cuda").to(dt(torch, dtype)))
    put(torch, c, r, seqs, counts, rows, layer)


def put(torch, c, r, seqs, counts, rows, layer=0):
    cu = np.concatenate([[0], np.cumsum(counts)])
    c.append(layer, rows[0], rows[1], seqs=ids(torch, seqs), cu=ids(torch, cu), n=max(max(counts), 1))
    host = [x.float().cpu().numpy() for x in rows]
    r.append(layer, seqs, *[[x[cu[i]:cu[i + 1]] for i in range(len(seqs))] for x in host])


def same(torch, c, r):
    """Tables, counts, and every held token's codes and scales, bit for bit."""
    assert np.array_equal(c.table.cpu().numpy(), r.table)
    assert np.array_equal(c.length.cpu().numpy(), r.length)
    assert np.array_equal(c.refs.cpu().numpy(), r.refs)
    got = [(c.k.cpu().numpy(), c.k_scale.cpu().numpy()), (c.v.cpu().numpy(), c.v_scale.cpu().numpy())]
    for s in range(r.n_seqs):
        for j, p in enumerate(r.table[s]):
            if p < 0:
                continue
            u = min(r.page, int(r.length[s]) - j * r.page)
            nb = -(-u // r.block)
            for z in range(2):
                assert np.array_equal(got[z][0][:, p, :, :u], r.codes[z, :, p, :, :u]), (s, j, z)
                assert np.array_equal(got[z][1][:, p, :, :nb], r.scale[z, :, p, :, :nb]), (s, j, z)


def check_attend(torch, c, r, seqs, counts, heads, dtype, rng, window=0, sinks=0, q=None, layer=0, qsize=1.5, **kw):
    cu = np.concatenate([[0], np.cumsum(counts)])
    if q is None:
        q = torch.tensor(rng.standard_normal((sum(counts), heads, r.d)) * qsize, dtype=torch.float32, device="cuda")
        q = q.to(dt(torch, dtype))
    scale = r.d ** -0.5
    out, lse = c.attend(layer, q, seqs=ids(torch, seqs), cu=ids(torch, cu), n=max(max(counts), 1), window=window,
                        sinks=sinks, return_lse=True, **kw)
    c.check()
    assert out.dtype == q.dtype
    got, z = out.float().cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    qh = q.float().cpu().numpy().astype(np.float64)
    u = 2.0 ** -24
    wt, rnd = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11, torch.finfo(q.dtype).eps / 2
    for i, s in enumerate(seqs):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        ref, rl, size, top = r.attend(layer, s, qh[a:b], scale, window, sinks)
        ds = size * (2.0 ** -22 + 2 * r.d * u) + 2.0 ** -21 * (size + 8)
        n = int(r.length[s])
        tol = top * (np.exp(2 * ds) - 1 + wt + 2.0 ** -18 + n * 2.0 ** -32)
        # what passes the type's largest value is infinite
        far = np.isinf(got[a:b]) & (np.abs(ref) * (1 + rnd) + tol[..., None] > torch.finfo(q.dtype).max)
        assert np.array_equal(np.sign(got[a:b][far]), np.sign(ref[far]))
        err = np.abs(np.where(far, ref, got[a:b]) - ref)
        assert np.all(err <= tol[..., None] + rnd * np.abs(ref) + 1e-37), (s, float((err - tol[..., None]).max()))
        none = np.isneginf(rl)
        assert np.array_equal(np.isneginf(z[a:b]), none) and not got[a:b][none].any()
        assert np.all(np.abs(z[a:b][~none] - rl[~none]) <= (ds + 2.0 ** -18 + 2.0 ** -21 * np.abs(rl))[~none])
    return out, lse


# ---- append and rows -------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,page,block", [(64, 16, 16), (128, 64, 32), (64, 48, 16), (128, 128, 64)])
def test_append_bit_exact(torch, dtype, d, page, block):
    rng = np.random.default_rng(d + page)
    c, r = make(torch, n_layers=2, d=d, page=page, block=block, kv=3, n_seqs=5, max_pages=6, n_pages=30)
    lens = [1, block, page + 3, 2 * page + block // 2 + 1]
    fill(torch, c, r, [3, 0, 4, 1], lens, rng, dtype, layer=1)
    same_layer(torch, c, r)
    # single tokens of growing size: the block's older codes are rounded again
    for step in range(5):
        fill(torch, c, r, [1, 3, 0], [1, 1, 1], rng, dtype, size=2.0 ** step, layer=1)
    # uneven chunks, one of them empty, over block and page borders
    fill(torch, c, r, [0, 2, 3, 1], [block + 5, page, 0, 7], rng, dtype, layer=1)
    same_layer(torch, c, r)
    c.check()


def same_layer(torch, c, r):
    """same() where only layer 1 was written: layer 0 of both is made equal first."""
    r.codes[0, 0], r.codes[1, 0] = c.k[0].cpu().numpy(), c.v[0].cpu().numpy()
    r.scale[0, 0], r.scale[1, 0] = c.k_scale[0].cpu().numpy(), c.v_scale[0].cpu().numpy()
    same2(torch, c, r)


def same2(torch, c, r):
    for t in (c.k_scale, c.v_scale):
        t[0].nan_to_num_(0.0)
    r.scale[:, 0] = np.nan_to_num(r.scale[:, 0], nan=0.0)
    same(torch, c, r)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 9, 16, 17, 40, 130])
def test_append_any_start(torch, n):
    rng = np.random.default_rng(n)
    c, r = make(torch, d=128, page=64, block=32, kv=2, n_seqs=4, max_pages=8, n_pages=32)
    for past in (0, 1, 31, 32):
        fill(torch, c, r, [past % 4 if past < 31 else past - 29], [max(past, 1)], rng)
    fill(torch, c, r, [0, 1, 2, 3], [n, n, n, n], rng)
    same(torch, c, r)


def test_append_strided_rows_of_a_fused_projection(torch):
    rng = np.random.default_rng(5)
    c, r = make(torch, d=64, kv=2, page=32, block=32)
    qkv = torch.tensor(rng.standard_normal((9, 6 + 2 + 2, 64)), dtype=torch.float32, device="cuda")
    assert r.reserve([0], [9])
    c.reserve(ids(torch, [9]), seqs=ids(torch, [0]))
    put(torch, c, r, [0], [9], [qkv[:, 6:8], qkv[:, 8:10]])
    same(torch, c, r)
    # head-major rows
    t = torch.tensor(rng.standard_normal((2, 5, 64)), dtype=torch.float32, device="cuda")
    assert r.reserve([1], [5])
    c.reserve(ids(torch, [5]), seqs=ids(torch, [1]))
    put(torch, c, r, [1], [5], [t.transpose(0, 1), t.transpose(0, 1) * 2])
    same(torch, c, r)


def test_append_values_that_are_not_finite_and_blocks_of_zeros(torch):
    rng = np.random.default_rng(6)
    c, r = make(torch, d=64, kv=1, page=16, block=16)
    x = rng.standard_normal((48, 1, 64)).astype(np.float32)
    x[3, 0, 5], x[4, 0, 6], x[5, 0, 7] = np.nan, np.inf, -np.inf
    x[16:32] = 0.0  # a block of zeros
    x[32:] *= 1e-36  # below what a scale holds
    x[40, 0, 0] = np.inf
    assert r.reserve([0], [48])
    c.reserve(ids(torch, [48]), seqs=ids(torch, [0]))
    rows = [torch.tensor(x, device="cuda")] * 2
    put(torch, c, r, [0], [48], rows)
    same(torch, c, r)
    k, v = c.rows(0, seqs=ids(torch, [0]), n=48)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    assert float(k[3, 0, 5]) == 0.0 and not k[16:32].any() and not k[32:].any()
    assert float(k[4, 0, 6]) == -float(k[5, 0, 7]) > 0
    # growth from a block of zeros, and sizes at both ends of f32
    y = np.zeros((2, 1, 64), np.float32)
    y[0, 0, 0], y[1, 0, 1] = 3e38, 1e-20
    assert r.reserve([1], [2])
    c.reserve(ids(torch, [2]), seqs=ids(torch, [1]))
    put(torch, c, r, [1], [2], [torch.tensor(y, device="cuda")] * 2)
    same(torch, c, r)
    check_attend(torch, c, r, [0], [2], 1, "f32", rng)


def test_rows_values_and_missing_tokens(torch):
    rng = np.random.default_rng(7)
    c, r = make(torch, d=64, kv=2, page=16, block=16, n_seqs=3)
    fill(torch, c, r, [0, 2], [40, 5], rng)
    for dtype in ("f32", "f16", "bf16"):
        # three more rows than sequence 2 holds: they read as zeros
        k, v = c.rows(0, seqs=ids(torch, [2, 0]), cu=ids(torch, [0, 8, 30]), n=22, total=30, dtype=dt(torch, dtype))
        for z, got in enumerate((k, v)):
            want = np.concatenate([np.zeros((3, 2, 64)), r.values(0, 2, z), r.values(0, 0, z)[18:]])
            want = torch.tensor(want.astype(np.float32)).to(dt(torch, dtype))
            assert torch.equal(got.cpu(), want)
    c.slide(8, 0, seqs=ids(torch, [0]))
    r.slide(8, 0, [0])
    k, _ = c.rows(0, seqs=ids(torch, [0]), n=40)
    assert not k[:32].any() and k[32:].any()
    c.check()


# ---- attention -----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 4), (3, 5), (2, 8), (1, 16), (2, 9), (1, 40)])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_heads(torch, dtype, kv, group, d):
    rng = np.random.default_rng(kv * 100 + group)
    c, r = make(torch, d=d, kv=kv, page=32, block=16, n_seqs=4, max_pages=12)
    fill(torch, c, r, [0, 1, 2], [1, 77, 300], rng, dtype)
    check_attend(torch, c, r, [0, 1, 2], [1, 1, 1], kv * group, dtype, rng)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 700])
@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (64, 64), (256, 32)])
def test_attend_lengths(torch, length, page, block):
    rng = np.random.default_rng(length)
    c, r = make(torch, d=64, kv=2, page=page, block=block, n_seqs=2, max_pages=-(-701 // page), n_pages=60)
    fill(torch, c, r, [1], [length], rng)
    n = min(length, 5)
    check_attend(torch, c, r, [1], [n], 4, "f32", rng)
    check_attend(torch, c, r, [1], [1], 4, "bf16", rng)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [2, 7, 16, 17, 33, 64, 100, 129, 260])
def test_attend_chunks(torch, dtype, n):
    rng = np.random.default_rng(n)
    c, r = make(torch, d=128, kv=2, page=64, block=32, n_seqs=3, max_pages=12)
    lens = [n, n + 1, n + 200]
    fill(torch, c, r, [0, 1, 2], lens, rng, dtype)
    check_attend(torch, c, r, [2, 0, 1], [n, n, max(1, n // 3)], 4, dtype, rng)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 100), (64, 16), (100, 0), (130, 65), (400, 3),
                                          (5000, 5), (1, 5000)])
@pytest.mark.parametrize("n", [1, 6, 70, 300])
def test_attend_window_and_sinks(torch, window, sinks, n):
    rng = np.random.default_rng(window * 7 + sinks + n)
    c, r = make(torch, d=64, kv=1, page=32, block=32, n_seqs=3, max_pages=20, n_pages=60)
    fill(torch, c, r, [0, 1, 2], [n, n + 31, n + 250], rng)
    for dtype in ("f32", "bf16"):
        check_attend(torch, c, r, [0, 1, 2], [n, n, n], 3, dtype, rng, window=window, sinks=sinks)
    # what slid out of the window takes no part and its pages may be anybody's
    c.slide(window, sinks)
    r.slide(window, sinks, range(3))
    check_attend(torch, c, r, [0, 1, 2], [1, 1, 1], 3, "f32", rng, window=window, sinks=sinks)
    check_attend(torch, c, r, [0, 1, 2], [n, n, n], 3, "f16", rng)  # the pages that are left, no window
    same(torch, c, r)


def test_attend_rows_that_see_nothing(torch):
    rng = np.random.default_rng(11)
    c, r = make(torch, d=64, kv=2, page=16, block=16, n_seqs=4)
    fill(torch, c, r, [0, 2], [3, 90], rng)
    # an empty sequence, more rows than tokens, no rows at all
    check_attend(torch, c, r, [1, 0, 2, 3], [2, 7, 0, 1], 4, "f32", rng)
    check_attend(torch, c, r, [1, 0, 2, 3], [40, 70, 33, 0], 4, "bf16", rng)
    # every page of a sequence is gone
    c.table[2] = -1
    r.table[2] = -1
    out, lse = check_attend(torch, c, r, [2], [5], 4, "f32", rng)
    assert not out.any() and torch.isneginf(lse).all()


def test_attend_sequences_outside_the_cache(torch):
    from stealcode_b200._lib import ScError

    rng = np.random.default_rng(12)
    c, r = make(torch, d=64, kv=1)
    fill(torch, c, r, [0], [9], rng)
    q = torch.ones(3, 2, 64, device="cuda")
    out = c.attend(0, q, seqs=ids(torch, [7, 0, -1]), n=1)
    assert not out[0].any() and out[1].any() and not out[2].any()
    c.append(0, torch.ones(1, 1, 64, device="cuda"), torch.ones(1, 1, 64, device="cuda"), seqs=ids(torch, [99]), n=1)
    with pytest.raises(ScError, match="sequence id"):
        c.check()
    c.clear_status()
    # page ids outside the pool are not followed
    c.table[0, 0] = 12345
    assert not c.attend(0, q[:1], seqs=ids(torch, [0]), n=1).any()
    with pytest.raises(ScError, match="page id"):
        c.check()
    # cu that leads outside the packed rows
    c.clear_status()
    c.table[0] = ids(torch, r.table[0])
    cu = ids(torch, [0, 2, 1000000])
    c.attend(0, q, seqs=ids(torch, [0, 1]), cu=cu, n=2000000 // 4)
    c.append(0, torch.ones(3, 1, 64, device="cuda"), torch.ones(3, 1, 64, device="cuda"), seqs=ids(torch, [1, 0]),
             cu=ids(torch, [-5, 2, -7]), n=4)
    torch.cuda.synchronize()


def test_attend_scores_and_scales_of_any_size(torch):
    rng = np.random.default_rng(13)
    c, r = make(torch, d=128, kv=1, page=32, block=16, n_seqs=4, max_pages=12)
    # value blocks between 2^-20 and 2^20, keys that grow: the running maximum moves in every tile
    n = 300
    x = rng.standard_normal((n, 1, 128)).astype(np.float32)
    grow = np.linspace(0.01, 4, n).astype(np.float32)[:, None, None]
    vs = np.exp2(rng.integers(-20, 21, n // 16 + 1)).astype(np.float32).repeat(16)[:n, None, None]
    assert r.reserve([0], [n])
    c.reserve(ids(torch, [n]), seqs=ids(torch, [0]))
    put(torch, c, r, [0], [n], [torch.tensor(x * grow, device="cuda"), torch.tensor(x * vs, device="cuda")])
    for dtype in ("f32", "f16", "bf16"):
        for size in (1e-4, 1.0, 20.0):
            check_attend(torch, c, r, [0], [3], 4, dtype, rng, qsize=size)
    # a row of q that is not finite spoils itself only
    q = torch.tensor(rng.standard_normal((3, 4, 128)), dtype=torch.float32, device="cuda")
    clean = c.attend(0, q, seqs=ids(torch, [0]), n=3)
    q2 = q.clone()
    q2[1, 2, 5], q2[2, 0, 0] = float("nan"), float("inf")
    got = c.attend(0, q2, seqs=ids(torch, [0]), n=3)
    assert torch.isnan(got[1, 2]).all() and torch.isnan(got[2, 0]).all()
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1, 2] = keep[2, 0] = False
    assert torch.equal(got[keep], clean[keep])
    # zeros: every key weighs the same
    check_attend(torch, c, r, [0], [2], 4, "f32", rng, q=torch.zeros(2, 4, 128, device="cuda"))


def test_attend_strides_layers_out_and_streams(torch):
    rng = np.random.default_rng(14)
    c, r = make(torch, n_layers=3, d=64, kv=2, page=32, block=16, n_seqs=2, max_pages=8)
    fill(torch, c, r, [0], [100], rng, layer=2)
    for dtype in ("f32", "bf16"):
        # q inside a fused projection; head-major q; out inside a wider tensor
        t = torch.tensor(rng.standard_normal((7, 10, 64)), dtype=torch.float32, device="cuda").to(dt(torch, dtype))
        check_attend(torch, c, r, [0], [7], 6, dtype, rng, q=t[:, 1:7], layer=2)
        hm = t[:, :4].transpose(0, 1).contiguous().transpose(0, 1)
        wide = torch.zeros(7, 8, 64, dtype=t.dtype, device="cuda")
        check_attend(torch, c, r, [0], [7], 4, dtype, rng, q=hm, out=wide[:, 2:6], layer=2)
        assert not wide[:, :2].any() and not wide[:, 6:].any()
        # odd element offsets (no 16-byte alignment)
        flat = torch.tensor(rng.standard_normal(7 * 5 * 64 + 3), dtype=torch.float32, device="cuda").to(t.dtype)
        check_attend(torch, c, r, [0], [7], 4, dtype, rng, q=flat[3:].view(7, 5, 64)[:, 1:], layer=2)
    q = torch.tensor(rng.standard_normal((7, 4, 64)), dtype=torch.float32, device="cuda")
    want = c.attend(2, q, seqs=ids(torch, [0]), n=7)
    side = torch.cuda.Stream()
    seqs = ids(torch, [0])
    torch.cuda.synchronize()
    got = c.attend(2, q, seqs=seqs, n=7, stream=side)
    with torch.cuda.stream(side):
        got2 = c.attend(2, q, seqs=seqs, n=7)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got2, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 20])
def test_attend_split_over_a_long_past(torch, dtype, n):
    rng = np.random.default_rng(15)
    c, r = make(torch, d=64, kv=1, page=64, block=64, n_seqs=3, max_pages=80, n_pages=200)
    fill(torch, c, r, [0, 1, 2], [5000, 33, 2100], rng)
    a = check_attend(torch, c, r, [0, 1, 2], [n, n, n], 8, dtype, rng)
    rng2 = np.random.default_rng(99)
    q = torch.tensor(rng2.standard_normal((3 * n, 8, 64)), dtype=torch.float32, device="cuda").to(dt(torch, dtype))
    first = c.attend(0, q, n=n, return_lse=True)
    for _ in range(5):  # the same bits, whichever block joins the parts
        again = c.attend(0, q, n=n, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    del a


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_long_chunks_without_alignment(torch, dtype, d):
    """Rows and results at odd element offsets, through the many-row kernel and the block-wise append; one
    sequence long enough that its items are split."""
    rng = np.random.default_rng(d)
    c, r = make(torch, d=d, kv=2, page=48, block=16, n_seqs=2, max_pages=40, n_pages=90)
    for s, n in ((0, 90), (1, 1500)):
        assert r.reserve([s], [n])
        c.reserve(ids(torch, [n]), seqs=ids(torch, [s]))
        flat = torch.tensor(rng.standard_normal(n * 5 * d + 3), dtype=torch.float32, device="cuda").to(dt(torch, dtype))
        kv = flat[3:].view(n, 5, d)
        put(torch, c, r, [s], [n], [kv[:, 1:3], kv[:, 3:5]])
    same(torch, c, r)
    flat = torch.tensor(rng.standard_normal(180 * 7 * d + 1), dtype=torch.float32, device="cuda").to(dt(torch, dtype))
    q = flat[1:].view(180, 7, d)[:, 1:]
    out = torch.zeros(180 * 8 * d + 1, dtype=q.dtype, device="cuda")[1:].view(180, 8, d)
    check_attend(torch, c, r, [1, 0], [90, 90], 6, dtype, rng, q=q, out=out[:, 1:7])
    assert not out[:, 0].any() and not out[:, 7].any()
    # scores turned round, and all alike
    for scale in (-0.3, 0.0):
        w = torch.zeros(180, 6, d, dtype=q.dtype, device="cuda")
        w.copy_(q)
        a, la = c.attend(0, w, seqs=ids(torch, [1, 0]), n=90, scale=scale, return_lse=True)
        b, lb = c.attend(0, w * -1 if scale else w * 0, seqs=ids(torch, [1, 0]), n=90, scale=-scale or 1.0, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("n", [1, 60])
def test_offsets_beyond_32_bits(torch, n):
    """Pages whose codes start beyond 2^32 bytes: the same bits as from a small pool."""
    from stealcode_b200 import KvCache8

    pages, used = 70000, 12
    big = KvCache8(1, pages, 8, 128, 2, 8, page=64, block=32)  # 64 KB a page
    small = KvCache8(1, used, 8, 128, 2, 8, page=64, block=32)
    big.refs[:pages - used] = 1  # in use by others
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(500, 8, 128, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(2 * n, 16, 128, generator=g, device="cuda")
    got = []
    for c in (big, small):
        c.reserve(ids(torch, [330, 170]))
        c.append(0, k, v, cu=ids(torch, [0, 330, 500]), n=330)
        out = c.attend(0, q, n=n, max_len=330)
        rows = c.rows(0, cu=ids(torch, [0, 330, 500]), n=330, total=500)
        c.release(ids(torch, [0]))
        c.fork(ids(torch, [1]), ids(torch, [0]))
        out2 = c.attend(0, q, n=n, max_len=330)
        c.check()
        got.append((out, out2) + rows)
    assert int(big.table.max()) == int(small.table.max()) + pages - used
    assert int(big.table[1, 0]) * 65536 > 2 ** 32
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_attend_in_a_cuda_graph(torch):
    rng = np.random.default_rng(16)
    c, r = make(torch, d=128, kv=2, page=32, block=16, n_seqs=2, max_pages=8)
    fill(torch, c, r, [0, 1], [60, 100], rng)
    q = torch.tensor(rng.standard_normal((2, 4, 128)), dtype=torch.float32, device="cuda")
    k = torch.tensor(rng.standard_normal((2, 2, 128)), dtype=torch.float32, device="cuda")
    one = ids(torch, [1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the workspaces of this stream
        c.attend(0, q, n=1)
        c.reserve(torch.zeros_like(one))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.reserve(one)
        c.append(0, k, k, n=1)
        out = c.attend(0, q, n=1)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert r.reserve([0, 1], [1, 1])
        kh = k.cpu().numpy()
        r.append(0, [0, 1], [kh[:1], kh[1:]], [kh[:1], kh[1:]])
        same(torch, c, r)
        assert torch.equal(out, c.attend(0, q, n=1))
    check_attend(torch, c, r, [0, 1], [1, 1], 4, "f32", rng, q=q)
    del g
    # a capture on a stream that has no workspace yet is refused
    h, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(h, stream=other):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before a graph capture"):
            c.attend(0, q, n=1)
    h.replay()
    torch.cuda.synchronize()
    assert bool((x == 1).all())
    del h


# ---- pages ---------------------------------------------------------------------------


@pytest.mark.parametrize("seed", range(4))
def test_pages_random_programs(torch, seed):
    """reserve, append, fork, release, slide and compact in a random order, step by step as the model."""
    rng = np.random.default_rng(seed)
    page, block = [(16, 16), (32, 16), (64, 32), (48, 16)][seed]
    c, r = make(torch, n_layers=2, d=64, kv=1, n_seqs=9, n_pages=60, max_pages=7, page=page, block=block, seed=seed)
    for t in (c.k_scale, c.v_scale):
        t.nan_to_num_(0.0)
    r.codes[0], r.codes[1] = c.k.cpu().numpy(), c.v.cpu().numpy()
    r.scale[0], r.scale[1] = c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy()
    for step in range(40):
        op = rng.choice(["fill", "fill", "fork", "release", "slide", "compact"])
        m = int(rng.integers(1, 6))
        seqs = [int(x) for x in rng.permutation(9)[:m]]
        if op == "fill":
            counts = [int(rng.integers(0, 2 * page)) if r.length[s] < 5 * page else 0 for s in seqs]
            free = int((r.refs == 0).sum())
            if sum(-(-x // page) + 1 for x in counts) > free:
                continue
            fill(torch, c, r, seqs, counts, rng, layer=0)
            put(torch, c, r, seqs, counts, [torch.tensor(rng.standard_normal((sum(counts), 1, 64)), dtype=torch.float32,
                                                         device="cuda") for _ in range(2)], layer=1)
        elif op == "fork":
            parents = [int(x) for x in rng.integers(0, 9, m)]
            if m > int((r.refs == 0).sum()):
                continue
            assert r.fork(parents, seqs)
            c.fork(ids(torch, parents), ids(torch, seqs))
        elif op == "release":
            r.release(seqs[:2])
            c.release(ids(torch, seqs[:2]))
        elif op == "slide":
            w, k = int(rng.integers(1, 3 * page)), int(rng.integers(0, 2 * page))
            r.slide(w, k, seqs)
            c.slide(w, k, seqs=ids(torch, seqs))
        else:
            r.compact()
            c.compact()
        c.check()
        same(torch, c, r)
        count = np.bincount(r.table[r.table >= 0], minlength=60)
        assert np.array_equal(count, r.refs)
    seqs = [s for s in range(9) if r.length[s] > 0]
    if seqs:
        check_attend(torch, c, r, seqs, [1] * len(seqs), 2, "f32", rng)


def test_pages_large_pool(torch):
    """More pages than one pass of the cluster over the pool takes."""
    n_pages, n_seqs = 50000, 300
    c, r = make(torch, d=64, kv=1, n_seqs=n_seqs, n_pages=n_pages, max_pages=128, page=16, block=16)
    for t in (c.k_scale, c.v_scale):
        t.nan_to_num_(0.0)
    r.codes[0], r.codes[1] = c.k.cpu().numpy(), c.v.cpu().numpy()
    r.scale[0], r.scale[1] = c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy()
    rng = np.random.default_rng(3)
    counts = rng.integers(0, 2000, n_seqs).tolist()
    assert r.reserve(range(n_seqs), counts)
    c.reserve(ids(torch, counts))
    gone = rng.permutation(n_seqs)[:150].tolist()
    r.release(gone)
    c.release(ids(torch, gone))
    r.compact()
    c.compact()
    same(torch, c, r)
    counts = rng.integers(0, 2000, 150).tolist()
    assert r.reserve(gone, counts)
    c.reserve(ids(torch, counts), seqs=ids(torch, gone))
    c.check()
    same(torch, c, r)


def test_pages_failures_change_nothing(torch):
    from stealcode_b200._lib import SC_ERR_ALLOC, SC_ERR_INVALID, ScError

    rng = np.random.default_rng(4)
    c, r = make(torch, d=64, kv=1, n_seqs=4, n_pages=6, max_pages=4, page=16, block=16)
    fill(torch, c, r, [0, 1], [20, 30], rng)

    def fails(code, call):
        call()
        # later calls that would change the cache do nothing
        c.reserve(ids(torch, [1]), seqs=ids(torch, [0]))
        c.append(0, torch.ones(1, 1, 64, device="cuda"), torch.ones(1, 1, 64, device="cuda"), seqs=ids(torch, [0]), n=1)
        c.fork(ids(torch, [0]), ids(torch, [3]))
        c.compact()
        with pytest.raises(ScError) as e:
            c.check()
        assert e.value.code == code
        same(torch, c, r)
        c.clear_status()

    fails(SC_ERR_ALLOC, lambda: c.reserve(ids(torch, [33, 16]), seqs=ids(torch, [2, 3])))  # 5 pages, 2 free
    fails(SC_ERR_ALLOC, lambda: c.reserve(ids(torch, [45]), seqs=ids(torch, [0])))  # 65 tokens, 4 pages of 16
    fails(SC_ERR_ALLOC, lambda: c.reserve(ids(torch, [2 ** 31 - 1]), seqs=ids(torch, [0])))
    fails(SC_ERR_INVALID, lambda: c.reserve(ids(torch, [1, 1]), seqs=ids(torch, [2, 2])))
    fails(SC_ERR_INVALID, lambda: c.reserve(ids(torch, [1]), seqs=ids(torch, [4])))
    fails(SC_ERR_INVALID, lambda: c.reserve(ids(torch, [-1]), seqs=ids(torch, [0])))
    fails(SC_ERR_INVALID, lambda: c.fork(ids(torch, [0, 1]), ids(torch, [2, 2])))
    fails(SC_ERR_INVALID, lambda: c.fork(ids(torch, [-1]), ids(torch, [2])))
    fails(SC_ERR_INVALID, lambda: c.fork(ids(torch, [0]), ids(torch, [17])))
    # the pool's last two pages go to two forks, a third finds none
    assert r.fork([0, 1], [2, 3])
    c.fork(ids(torch, [0, 1]), ids(torch, [2, 3]))
    same(torch, c, r)
    fails(SC_ERR_ALLOC, lambda: c.fork(ids(torch, [0]), ids(torch, [1])))
    # giving pages back is how a caller recovers: release runs while a bit is set
    fill(torch, c, r, [1], [2], rng)
    c.reserve(ids(torch, [17]), seqs=ids(torch, [1]))
    c.release(ids(torch, [2, 2]))
    r.release([2])
    with pytest.raises(ScError):
        c.check()
    same(torch, c, r)
    c.clear_status()
    # an append without a reserved page
    c.length[0] += 20
    c.append(0, torch.ones(20, 1, 64, device="cuda"), torch.ones(20, 1, 64, device="cuda"), seqs=ids(torch, [0]), n=20)
    with pytest.raises(ScError, match="page id"):
        c.check()


# ---- the whole step -------------------------------------------------------------------


def test_arguments_are_refused(torch):
    from stealcode_b200 import KvCache8
    from stealcode_b200._lib import SC_ERR_INVALID, SC_ERR_UNSUPPORTED, ScError

    c, _ = make(torch, d=64, kv=2)
    q = torch.zeros(4, 4, 64, device="cuda")
    kv = torch.zeros(4, 2, 64, device="cuda")
    bad = [
        lambda: c.attend(0, q.double(), n=1),
        lambda: c.attend(0, q[..., :32], n=1),
        lambda: c.attend(0, q.transpose(1, 2).contiguous().transpose(1, 2), n=1),
        lambda: c.attend(0, q.cpu(), n=1),
        lambda: c.attend(0, q),
        lambda: c.attend(0, q, n=1, out=torch.zeros(4, 4, 64, device="cuda", dtype=torch.float16)),
        lambda: c.attend(0, q, seqs=torch.zeros(4, dtype=torch.int64, device="cuda"), n=1),
        lambda: c.attend(0, q, seqs=ids(torch, [0, 1]), cu=ids(torch, [0, 1]), n=1),
        lambda: c.append(0, kv, kv.half(), n=1),
        lambda: c.append(0, kv, kv[:3], n=1),
        lambda: c.append(0, q, q, n=1),
        lambda: c.rows(0, cu=ids(torch, [0, 1]), n=1),
        lambda: c.rows(0, n=1, dtype=torch.int8),
        lambda: c.reserve(ids(torch, [1, 2]), seqs=ids(torch, [1])),
        lambda: c.fork(ids(torch, [1, 2]), ids(torch, [1])),
        lambda: KvCache8(1, 4, 1, 64, 1, 4, page=30, block=16),
        lambda: KvCache8.wrap(c.k, c.v, c.k_scale, c.v_scale, c.table.long(), c.length, c.refs),
        lambda: KvCache8.wrap(c.k, c.v, c.k_scale, c.v_scale, c.table, c.length, c.refs[1:]),
        lambda: KvCache8.wrap(c.k.transpose(2, 3), c.v.transpose(2, 3), c.k_scale, c.v_scale, c.table, c.length, c.refs),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(i)
    for call in (lambda: c.attend(1, q, n=1), lambda: c.attend(-1, q, n=1), lambda: c.attend(0, q[:, :3], n=1),
                 lambda: c.attend(0, q, n=1, window=-1), lambda: c.attend(0, q, n=1, sinks=-1),
                 lambda: c.attend(0, q, n=3), lambda: c.slide(0), lambda: c.append(0, kv, kv, n=3)):
        with pytest.raises(ScError) as e:
            call()
        assert e.value.code == SC_ERR_INVALID
    for shape, page, block in ((80, 32, 16), (64, 8, 8), (64, 2048, 16), (64, 128, 128)):
        odd = KvCache8(1, 4, 1, shape, 1, 4, page=page, block=block)
        with pytest.raises(ScError) as e:
            odd.attend(0, torch.zeros(1, 1, shape, device="cuda"), n=1)
        assert e.value.code == SC_ERR_UNSUPPORTED
    # nothing to do is no error
    c.append(0, kv[:0], kv[:0], seqs=ids(torch, []), n=1)
    assert c.attend(0, q[:0], seqs=ids(torch, []), n=1).shape == (0, 4, 64)
    c.reserve(ids(torch, []), seqs=ids(torch, []))
    c.release(ids(torch, []))
    c.check()
