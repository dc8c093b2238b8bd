"""GPU tests of the paged 8-bit cache's calls on a stream that is named in the
call: their inputs outlive the work, and a capture on that stream is seen."""
import numpy as np
import pytest

from tests.test_kv8_gpu import fill, ids, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t

    assert _t.cuda.is_available()
    return _t


def busy(torch, side):
    """Work of some milliseconds on a stream, so that what is queued there later starts late."""
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)


def test_inputs_of_a_call_on_another_stream_are_kept(torch):
    """Temporaries handed to a call with stream=: their memory is not given out again before the work has read it."""
    rng = np.random.default_rng(1)
    c, r = make(torch, d=128, kv=2, page=32, block=16, n_seqs=4, max_pages=40, n_pages=130)
    fill(torch, c, r, [0, 1], [300, 200], rng)
    side = torch.cuda.Stream()
    c.attend(0, torch.zeros(4, 4, 128, device="cuda"), n=1, stream=side)  # the stream's workspaces
    c.reserve(ids(torch, [0]), stream=side)
    torch.cuda.synchronize()
    src = torch.tensor(rng.standard_normal((256, 4, 128)), dtype=torch.float32, device="cuda").half()

    def reuse(shapes):  # whatever was freed meanwhile is handed out again and overwritten
        for shape, dtype in shapes:
            for _ in range(12):
                x = torch.empty(shape, dtype=dtype, device="cuda")
                x.fill_(3)
                hold.append(x)

    hold = []
    want = c.attend(0, src, seqs=ids(torch, [0, 1]), n=128)
    torch.cuda.synchronize()
    busy(torch, side)
    got = c.attend(0, src * 1, seqs=ids(torch, [0, 1]), n=128, stream=side)
    reuse([((256, 4, 128), torch.float16), (2, torch.int32)])
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # append and reserve: counts, rows, cu
    rows = [torch.tensor(rng.standard_normal((60, 2, 128)), dtype=torch.float32, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    busy(torch, side)
    c.reserve(ids(torch, [40, 20]), seqs=ids(torch, [2, 3]), stream=side)
    reuse([(2, torch.int32)])
    c.append(0, rows[0] * 1, rows[1] * 1, seqs=ids(torch, [2, 3]), cu=ids(torch, [0, 40, 60]), n=40, stream=side)
    reuse([((60, 2, 128), torch.float32), (2, torch.int32), (3, torch.int32)])
    torch.cuda.synchronize()
    c.check()
    assert r.reserve([2, 3], [40, 20])
    h = [x.cpu().numpy() for x in rows]
    r.append(0, [2, 3], *[[x[:40], x[40:]] for x in h])
    from tests.test_kv8_gpu import same

    same(torch, c, r)


def test_a_cache_outlives_its_work_on_another_stream(torch):
    """The cache is dropped while a call on another stream is queued: its memory is kept until that has run."""
    from stealcode_b200 import KvCache8

    side = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = torch.randn(200, 2, 64, generator=g, device="cuda")
    q = torch.randn(1, 4, 64, generator=g, device="cuda")
    got = []
    for late in (False, True):
        c = KvCache8(1, 64, 2, 64, 1, 64, page=16, block=16)
        c.reserve(ids(torch, [200]))
        c.append(0, rows, rows, n=200)
        c.attend(0, q, n=1, stream=side)
        shapes = [(t.shape, t.dtype) for t in (c.k, c.k_scale, c.table, c.length)]
        torch.cuda.synchronize()
        if late:
            busy(torch, side)
        got.append(c.attend(0, q, n=1, stream=side))
        del c
        hold = [torch.full(s, 1, dtype=d, device="cuda") for s, d in shapes for _ in range(4)]
        torch.cuda.synchronize()
        del hold
    assert torch.equal(got[0], got[1]) and got[0].any()


def test_a_capture_on_the_named_stream_is_refused(torch):
    """The stream of the call captures, the current one does not: no workspace is made inside the graph."""
    rng = np.random.default_rng(3)
    c, r = make(torch, d=64, kv=1)
    fill(torch, c, r, [0], [9], rng)
    q = torch.zeros(4, 2, 64, device="cuda")
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    refused = False
    with torch.cuda.graph(g, stream=side, capture_error_mode="relaxed"):
        x.add_(1)
        with torch.cuda.stream(other):
            try:
                c.attend(0, q, n=1, out=out, stream=side)
            except RuntimeError as e:
                refused = "before a graph capture" in str(e)
    g.replay()
    torch.cuda.synchronize()
    assert refused and bool((x == 1).all())
    del g
