"""GPU test of the attention inside the live-decoder example's step: every
layer's attention rows, before the output projection, against 64 bits over the
stored keys and values with a mask that the test makes from its own positions.

The bound is 1e-4 of the largest value (f32 rows: errors near 2^-18 of it); the
same comparison with a wrong mask, order or no attention has to be 20 times
over it, so that the test would see such a mistake."""
import numpy as np
import pytest
import torch

from tests.test_live_decoder_gpu import ex, small  # noqa: F401 (ex: the fixture)

pytestmark = pytest.mark.gpu

WINDOW, SINKS, PAGE = 40, 3, 16


def spy(cache):
    log, real = [], cache.attend

    def attend(layer, q, **kw):
        out = real(layer, q, **kw)
        log.append((layer, q.double().cpu().numpy(), out.double().cpu().numpy()))
        return out

    cache.attend = attend
    return log


def masks(p, length):
    t = np.arange(length)
    inside = (t > p - WINDOW) | (t < SINKS)
    return {"right": (t <= p) & inside, "not itself": (t < p) & inside, "one later": (t <= p) & ((t > p - WINDOW + 1) | (t < SINKS)),
            "no window": t <= p, "no sinks": (t <= p) & (t > p - WINDOW), "not causal": inside}


def compare(ex, dec, log, spans, controls=()):
    """spans: (sequence, its length before the step, its new tokens), in packed order; errors by kind of mask,
    as parts of the bound."""
    worst = dict.fromkeys(("right",) + tuple(controls), 0.0)
    heads, kv, hd = dec.heads, dec.kv, dec.hd
    for layer, q, out in log:
        row = 0
        for s, before, n in spans:
            length = before + n
            k, v = (x.double().cpu().numpy() for x in dec.cache.rows(layer, seqs=ex.ids([s]), n=length))
            bound = 1e-4 * np.abs(v).max()
            for i in range(n):
                for kind in worst:
                    see = masks(before + i, length)["right" if kind in ("none", "pages") else kind]
                    kk, vv = (np.roll(x, PAGE, 0) for x in (k, v)) if kind == "pages" else (k, v)
                    ref = np.zeros((heads, hd))
                    for h in range(heads):
                        if kind == "none" or not see.any():
                            continue
                        w = kk[see, h * kv // heads] @ q[row, h] * hd ** -0.5
                        w = np.exp(w - w.max())
                        ref[h] = (w / w.sum()) @ vv[see, h * kv // heads]
                    worst[kind] = max(worst[kind], np.abs(ref - out[row]).max() / bound)
                row += 1
        assert row == len(q)
    log.clear()
    return worst


def test_steps_attend_over_the_right_tokens(ex):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(5)
    dec = small(ex)
    log = spy(dec.cache)
    lens = {3: 0, 0: 0, 5: 0}

    def step(counts):
        seqs, n = list(counts), max(counts.values())
        cu = np.concatenate([[0], np.cumsum(list(counts.values()))])
        x = torch.randn(int(cu[-1]), 256, generator=g, device="cuda")
        dec.step(x, ex.ids(list(counts.values())), n, seqs=ex.ids(seqs), cu=ex.ids(cu))
        spans = [(s, lens[s], k) for s, k in counts.items()]
        for s, k in counts.items():
            lens[s] += k
        return spans

    kinds = ("not itself", "one later", "no window", "no sinks", "none", "pages")
    worst = compare(ex, dec, log, step({3: 70, 0: 23}), kinds + ("not causal",))
    assert worst.pop("right") <= 1.0
    assert min(worst.values()) >= 20.0, worst
    for _ in range(3):
        worst = compare(ex, dec, log, step({0: 1, 3: 1}), ())
        assert worst["right"] <= 1.0
    worst = compare(ex, dec, log, step({3: 1}), kinds)
    assert worst.pop("right") <= 1.0
    assert min(worst.values()) >= 20.0, worst
    # what left the window is given back, pages move, and the steps go on
    dec.tidy()
    dec.cache.compact()
    for counts in ({3: 9, 0: 1, 5: 17}, {5: 1, 3: 1}, {0: 30}):
        assert compare(ex, dec, log, step(counts))["right"] <= 1.0
    dec.cache.check()
