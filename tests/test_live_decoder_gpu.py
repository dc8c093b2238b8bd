"""GPU test of the live-decoder example: the 8-bit cache's operators in use,
held to what must not change a bit of the outputs (sharing a past, moving
pages, freeing what left the window) and to the same decoder with its keys
and values recomputed in one pass."""
import importlib.util
import os

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    import torch

    assert torch.cuda.is_available()
    spec = importlib.util.spec_from_file_location("live_decoder", os.path.join(ROOT, "examples", "live_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def small(ex, **kw):
    return ex.Decoder(layers=2, d_model=256, heads=4, kv_heads=2, d_ff=256, streams=6, pages=64, max_pages=16,
                      window=kw.pop("window", 40), sinks=3, page=16, block=16, **kw)


def feed(ex, dec, x, seqs, n):
    import torch

    return dec.step(x, ex.ids([n] * len(seqs)), n, seqs=ex.ids(seqs)) if len(seqs) else torch.empty(0, 256, device="cuda")


def test_forks_moves_and_slides_change_no_bit(ex):
    import torch

    g = torch.Generator(device="cuda").manual_seed(3)
    a, b = small(ex), small(ex)
    x = torch.randn(3 * 50, 256, generator=g, device="cuda")
    assert torch.equal(feed(ex, a, x, [0, 1, 2], 50), feed(ex, b, x, [0, 1, 2], 50))
    # b gives its old pages back, ends stream 0 and moves its pages together
    b.tidy()
    b.cache.release(ex.ids([0]))
    b.cache.compact()
    live = int((b.cache.refs > 0).sum())
    assert live < int((a.cache.refs > 0).sum()) and not b.cache.refs[live:].any()
    y = torch.randn(2, 256, generator=g, device="cuda")
    for _ in range(20):
        p, q = feed(ex, a, y, [1, 2], 1), feed(ex, b, y, [1, 2], 1)
        assert torch.equal(p, q)
        y = ex.norm(p)
    # children of stream 2 share its pages; in a copy of the decoder every page of theirs is a plain copy.
    # (The same call on the same lengths: how the work is cut, and so the rounding, depends on the batch.)
    d = small(ex)
    d.layers = b.layers
    for name in ("k", "v", "k_scale", "v_scale", "table", "length", "refs"):
        getattr(d.cache, name).copy_(getattr(b.cache, name))
    b.cache.fork(ex.ids([2, 2]), ex.ids([4, 5]))
    free = 63
    for child in (4, 5):
        for j, page in enumerate(d.cache.table[2].tolist()):
            if page >= 0:
                for name in ("k", "v", "k_scale", "v_scale"):
                    getattr(d.cache, name)[:, free] = getattr(d.cache, name)[:, page]
                d.cache.table[child, j] = free
                d.cache.refs[free] = 1
                free -= 1
        d.cache.length[child] = d.cache.length[2]
    assert int((b.cache.refs > 1).sum()) > 0 and int((d.cache.refs > 1).sum()) == 0
    for i in range(40):
        z = torch.randn(3, 256, generator=g, device="cuda")
        assert torch.equal(feed(ex, b, z, [5, 2, 4], 1), feed(ex, d, z, [5, 2, 4], 1))
    d.cache.check()
    a.cache.check()
    b.cache.check()


def test_step_by_step_is_the_prompt_at_once(ex):
    """Appending a prompt at once and token by token: blocks end with the same scales, so the stored values
    differ by the second rounding of older rows only (half a step of the final scale), and the outputs by
    what that and the values that a token saw before its block's later rows came do to a random decoder:
    a few per cent.  A wrong mask, position or page is off by the size of the output."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(70, 256, generator=g, device="cuda")
    a, b = small(ex), small(ex)
    whole = feed(ex, a, x, [3], 70)
    steps = torch.cat([feed(ex, b, x[i:i + 1], [3], 1) for i in range(70)])
    err = (whole - steps).norm() / whole.norm()
    assert err < 0.05, float(err)


def test_example_runs(ex):
    dec, x, y = ex.run(streams=8, layers=2, steps=70, d_model=256, heads=4, kv_heads=2, d_ff=256, window=64, sinks=4,
                       pages=256, prompt=(5, 200), quiet=True)
    import torch

    assert torch.isfinite(x).all() and torch.isfinite(y).all()
    live = int((dec.cache.refs > 0).sum())
    assert live and not dec.cache.refs[live:].any()
