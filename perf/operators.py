"""The operators of the paged 8-bit key/value cache, as they are measured.

Three operators share one cache (``stealcode_b200.KvCache8``): ``append``
(quantise new key/value rows into the pages, and read the stored values back),
``attend`` (attention over the pages, with an optional sliding window and first
tokens that stay visible) and the page operations (``fork``, ``compact`` and the
release / reserve / slide of streams that come and go).

Tensors of a state: ``k``, ``v`` int8 [layers, pages, kv_heads, page, head_dim];
``k_scale``, ``v_scale`` f32 [layers, pages, kv_heads, page / block]; ``table``
int32 [seqs, max_pages] (-1: none); ``length`` int32 [seqs]; ``refs`` int32 [pages].
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_TINY = 1e-30  # a block whose largest magnitude is below this is stored as zeros


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # One generated token of 64 live streams goes into the cache of a layer.
        dict(name="append step", op="append", m=64, n_lo=1, n_hi=1, len_lo=100, len_hi=4000, kv=8, d=128,
             page=64, block=32, dtype="bf16"),
        # Six prompts of uneven lengths, as the f32 projections of the framework give them.
        dict(name="append prompts", op="append", m=6, n_lo=37, n_hi=8192, len_lo=37, len_hi=8192, kv=8, d=128,
             page=64, block=64, dtype="f32"),
        # The smallest call: one live stream with a short past, one token, f32 (8 heads of 128).
        dict(name="attend one stream", op="attend", m=1, n_lo=1, n_hi=1, len_lo=500, len_hi=500, heads=8, kv=8,
             d=128, page=64, block=32, dtype="f32", window=0, sinks=0),
        # A batch of 64 streams of very uneven age, one token each, four query heads to a key head.
        dict(name="attend 64 streams", op="attend", m=64, n_lo=1, n_hi=1, len_lo=512, len_hi=16384, heads=32, kv=8,
             d=128, page=64, block=32, dtype="bf16", window=0, sinks=0),
        # 256 endless live streams in chunks of 7 frames: a window of 560 frames and 4 first frames, f32.
        dict(name="attend live window", op="attend", m=256, n_lo=7, n_hi=7, len_lo=50, len_hi=4000, heads=8, kv=8,
             d=128, page=16, block=16, dtype="f32", window=560, sinks=4),
        # A few very long recordings, one token each: the work is split over the long axis.
        dict(name="attend long past", op="attend", m=4, n_lo=1, n_hi=1, len_lo=65537, len_hi=131072, heads=32, kv=8,
             d=128, page=128, block=64, dtype="bf16", window=0, sinks=0),
        # A whole prompt at once.
        dict(name="attend prompt", op="attend", m=1, n_lo=4096, n_hi=4096, len_lo=4096, len_hi=4096, heads=32, kv=8,
             d=128, page=64, block=32, dtype="bf16", window=0, sinks=0),
        # Uneven chunks of prompts after a past, with a window and sinks, heads of 64.
        dict(name="attend chunks window", op="attend", m=4, n_lo=301, n_hi=1024, len_lo=5000, len_hi=12289, heads=16,
             kv=4, d=64, page=32, block=32, dtype="f16", window=2048, sinks=64),
        # 64 recordings of 750 frames, f32 (the framework's prefill batch).
        dict(name="attend prefill f32", op="attend", m=64, n_lo=750, n_hi=750, len_lo=750, len_hi=750, heads=8, kv=8,
             d=128, page=64, block=64, dtype="f32", window=0, sinks=0),
        # A beam step: 32 streams of 8 hypotheses each take over their parents' pasts, 24 layers.
        dict(name="pages fork", op="fork", m=32, beams=8, layers=24, len_lo=130, len_hi=700, kv=8, d=128, page=64,
             block=32, spare=1),
        # Half of the pool's streams have gone: the rest moves to the lowest pages, 24 layers.
        dict(name="pages compact", op="compact", m=128, layers=24, len_lo=100, len_hi=1500, kv=8, d=128, page=64,
             block=32),
        # 256 of 512 streams end, as many begin with a prompt, and what is outside the window is freed.
        dict(name="pages turnover", op="turnover", m=512, layers=1, len_lo=500, len_hi=8000, kv=1, d=64, page=16,
             block=16, window=1024, sinks=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges; none costs more than the largest listed one."""
    page = rng.choice([16, 32, 48, 64, 128])
    block = rng.choice([b for b in (16, 32, 64) if page % b == 0])
    c = dict(kv=rng.choice([1, 2, 3, 4, 8]), d=rng.choice([64, 128]), page=page, block=block)
    op = rng.choice(["append", "attend step", "attend step", "attend chunk", "attend prompt", "pages"])
    if op == "append":
        n_hi = _log(rng, 1, 4096)
        c.update(op="append", m=_log(rng, 1, max(1, min(256, 32768 // n_hi))), n_lo=rng.randint(1, n_hi), n_hi=n_hi,
                 dtype=rng.choice(["bf16", "f16", "f32"]))
        past = rng.choice([0, 0, _log(rng, 1, 2000)])
        c.update(len_lo=n_hi + past // 2, len_hi=n_hi + past)
        return c
    if op == "pages":
        kind = rng.choice(["fork", "compact", "turnover"])
        if kind == "fork":
            c.update(op="fork", m=_log(rng, 1, 32), beams=rng.randint(2, 8), layers=_log(rng, 1, 24))
            c.update(len_lo=_log(rng, 20, 300))
            c.update(len_hi=rng.randint(c["len_lo"], 700), spare=rng.randint(0, 40))
        elif kind == "compact":
            c.update(op="compact", m=_log(rng, 2, 128), layers=_log(rng, 1, 24), len_lo=_log(rng, 20, 500))
            c.update(len_hi=rng.randint(c["len_lo"], 1500))
        else:
            c.update(op="turnover", m=_log(rng, 2, 512), layers=1, kv=1, d=64, len_lo=_log(rng, 100, 2000))
            c.update(len_hi=rng.randint(c["len_lo"], 8000), window=_log(rng, 16, 2048), sinks=rng.choice([0, 4, 33]))
        return c
    group = rng.choice([1, 2, 4, 5, 8])
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 16, 4096), rng.choice([0, 1, 4, 64, 100]))])
    c.update(op="attend", heads=c["kv"] * group, dtype=rng.choice(["bf16", "f16", "f32"]), window=window, sinks=sinks)
    if op == "attend step":
        n = rng.choice([1, 1, 1, 2, 7])
        hi = _log(rng, n + 1, 65536)
        m = _log(rng, 1, max(1, min(256, (1 << 19) // max(hi, 512))))
        c.update(m=m, n_lo=n, n_hi=n, len_lo=max(n, _log(rng, max(n, hi // 20), hi)), len_hi=hi)
    elif op == "attend chunk":
        hi = _log(rng, 600, 12000)
        n_hi = _log(rng, 8, 512)
        c.update(m=rng.randint(1, 4), n_lo=rng.randint(1, n_hi), n_hi=n_hi, len_lo=rng.randint(n_hi, hi), len_hi=hi)
    else:
        n = _log(rng, 32, 3000)
        c.update(m=_log(rng, 1, max(1, min(64, (2500 * 2500) // (n * n)))), n_lo=n, n_hi=n, len_lo=n, len_hi=n)
    return c


def _spread(lo, hi, m):
    """m whole numbers spread over [lo, hi] by their logarithm, in an order of no pattern."""
    if m == 1:
        return [hi]
    v = [int(round(lo * (hi / lo) ** (i / (m - 1)))) for i in range(m)]
    step = next(s for s in range(max(1, int(m * 0.618)), 2 * m) if math.gcd(s, m) == 1)
    return [v[(i * step) % m] for i in range(m)]


def _lens(c):
    """(length after the call, new tokens) of every sequence of an append or attend case."""
    length, n = _spread(c["len_lo"], c["len_hi"], c["m"]), _spread(c["n_lo"], c["n_hi"], c["m"])
    if c["op"] == "append" and c["len_lo"] == c["n_lo"]:  # whole prompts
        length = n
    return length, [min(a, b) for a, b in zip(n, length)]


def _back(c):
    """Tokens of every sequence that an append may change: the new ones and the older ones of their first block."""
    return [b + (a - b) % c["block"] for a, b in zip(*_lens(c))]


def _starts(n):
    return torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32)


def _pages(length, page):
    return -(-length // page)


# ---- inputs --------------------------------------------------------------------


def _pool(gen, layers, n_pages, c, measured):
    """Codes and scales of a pool.  `measured`: quantised from keys with a few large channels and
    values of uneven size, as a model writes them; else any codes (they are only moved)."""
    kv, d, page, block = c["kv"], c["d"], c["page"], c["block"]
    dev = "cuda"
    out = []
    for which in range(2):
        codes = torch.empty(layers, n_pages, kv, page, d, dtype=torch.int8, device=dev)
        scale = torch.empty(layers, n_pages, kv, page // block, device=dev)
        if not measured:
            flat = codes.view(-1)
            for a in range(0, flat.numel(), 1 << 28):  # in parts, for memory
                part = flat[a:a + (1 << 28)]
                part.copy_(torch.randint(-127, 128, part.shape, generator=gen, device=dev, dtype=torch.int8))
            scale.copy_(torch.rand(scale.shape, generator=gen, device=dev) * 0.03 + 0.001)
            out += [codes, scale]
            continue
        chan = torch.exp(0.5 * torch.randn(kv, 1, 1, d, generator=gen, device=dev))
        chan = chan / chan.square().mean(-1, keepdim=True).sqrt()
        step = max(1, (1 << 26) // (kv * page * d))
        for a in range(0, n_pages, step):
            b = min(n_pages, a + step)
            x = torch.randn(b - a, kv, page // block, block, d, generator=gen, device=dev)
            x = x * chan if which == 0 else x * torch.exp(
                0.5 * torch.randn(b - a, kv, page // block, 1, 1, generator=gen, device=dev))
            s = x.abs().amax((-1, -2)) / 127
            scale[0, a:b] = s
            codes[0, a:b] = torch.round(x / s[..., None, None]).clamp_(-127, 127).reshape(b - a, kv, page, d)
        out += [codes, scale]
    return out[0], out[1], out[2], out[3]


def _table(gen, owned, n_pages, max_pages):
    """Page tables that hand out shuffled pages, and the pages' reference counts."""
    perm = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    count = torch.tensor(owned, device="cuda")
    at = torch.cumsum(count, 0) - count
    j = torch.arange(max_pages, device="cuda")
    use = j[None] < count[:, None]
    table = torch.where(use, perm[(at[:, None] + j).clamp_(max=n_pages - 1)], torch.full_like(perm[:1], -1))
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[table[use].long()] = 1
    return table.contiguous(), refs


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=c, op=c["op"], page=c["page"], block=c["block"])
    if c["op"] in ("append", "attend"):
        length, n = _lens(c)
        owned = [_pages(x, c["page"]) for x in length]
        n_pages, max_pages = sum(owned) + 3, max(owned)
        s["k"], s["k_scale"], s["v"], s["v_scale"] = _pool(gen, 1, n_pages, c, True)
        s["table"], s["refs"] = _table(gen, owned, n_pages, max_pages)
        s["length"] = torch.tensor(length, dtype=torch.int32, device="cuda")
        total, s["max_n"], s["max_len"] = sum(n), max(n), max(length)
        s["cu"] = None
        if min(n) != max(n):
            s["cu"] = _starts(n)
        dt = _DT[c["dtype"]]
        if c["op"] == "append":
            chan = torch.exp(0.5 * torch.randn(c["kv"], c["d"], generator=gen, device="cuda"))
            s["k_new"] = (torch.randn(total, c["kv"], c["d"], generator=gen, device="cuda") * chan).to(dt)
            s["v_new"] = torch.randn(total, c["kv"], c["d"], generator=gen, device="cuda").to(dt)
            back = _back(c)
            s["back"], s["max_back"], s["rows"] = _starts(back), max(back), sum(back)
        else:
            s["q"] = (1.5 * torch.randn(total, c["heads"], c["d"], generator=gen, device="cuda")).to(dt)
            s["window"], s["sinks"], s["scale"] = c["window"], c["sinks"], c["d"] ** -0.5
        return s
    if c["op"] == "fork":
        hyps = c["m"] * c["beams"]
        length = [x for x in _spread(c["len_lo"], c["len_hi"], c["m"]) for _ in range(c["beams"])]
        owned = [_pages(x, c["page"]) for x in length]
        # every hypothesis of a stream shares its full pages and has a last page of its own
        shared = [x // c["page"] for x in length]
        last = [a - b for a, b in zip(owned, shared)]
        n_pages = sum(shared[:: c["beams"]]) + 2 * sum(last) + c["spare"]
        s["k"], s["k_scale"], s["v"], s["v_scale"] = _pool(gen, c["layers"], n_pages, c, False)
        full, _ = _table(gen, [a + b * c["beams"] for a, b in zip(shared[:: c["beams"]], last[:: c["beams"]])], n_pages,
                         max(owned) + c["beams"])
        stream = torch.arange(hyps, device="cuda") // c["beams"]
        beam = torch.arange(hyps, device="cuda") % c["beams"]
        sh, la = (torch.tensor(x, device="cuda")[:, None] for x in (shared, last))
        j = torch.arange(max(owned), device="cuda")[None]
        src = torch.where(j < sh, j.expand(hyps, -1), sh + beam[:, None])
        t = torch.gather(full[stream], 1, src.clamp(max=full.shape[1] - 1))
        s["table"] = torch.where(j < sh + la, t, torch.full_like(t, -1)).contiguous()
        s["refs"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        ok = s["table"] >= 0
        s["refs"].scatter_add_(0, s["table"].clamp(min=0).long().flatten(), ok.int().flatten())
        s["length"] = torch.tensor(length, dtype=torch.int32, device="cuda")
        s["children"] = torch.arange(hyps, dtype=torch.int32, device="cuda")
        pick = torch.randint(0, c["beams"], (hyps,), generator=gen, device="cuda")
        s["parents"] = (stream * c["beams"] + pick).to(torch.int32)
        return s
    length = _spread(c["len_lo"], c["len_hi"], c["m"])
    owned = [_pages(x, c["page"]) for x in length]
    n_pages = sum(owned) + 5
    s["k"], s["k_scale"], s["v"], s["v_scale"] = _pool(gen, c["layers"], n_pages, c, False)
    s["table"], s["refs"] = _table(gen, owned, n_pages, max(owned))
    s["length"] = torch.tensor(length, dtype=torch.int32, device="cuda")
    gone = torch.arange(0, c["m"], 2, device="cuda")
    if c["op"] == "compact":  # every other stream has gone
        t = s["table"][gone]
        s["refs"][t[t >= 0].long()] = 0
        s["table"][gone] = -1
        s["length"][gone] = 0
        s["was"] = [s[x].clone() for x in ("table", "refs")]
    else:
        s["seqs"] = gone.to(torch.int32)
        s["counts"] = s["length"][gone].clone()
        s["window"], s["sinks"] = c["window"], c["sinks"]
    return s


# ---- the plain forms -------------------------------------------------------------


def _rows_of(s, n_each):
    """(sequence, index within its new tokens, new tokens of the sequence) of every packed row."""
    m = s["length"].shape[0]
    if s["cu"] is None:
        seq = torch.arange(m, device="cuda").repeat_interleave(n_each)
        return seq, torch.arange(m * n_each, device="cuda") % n_each, torch.full((m,), n_each, device="cuda")
    cu = s["cu"].long()
    total = s["k_new" if s["op"] == "append" else "q"].shape[0]
    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    return seq, t - cu[seq], cu[1:] - cu[:-1]


def _plain_append(s):
    page, block = s["page"], s["block"]
    seq, j, n = _rows_of(s, s["max_n"])
    length = s["length"].long()
    pos = length[seq] - n[seq] + j
    pg, slot = s["table"][seq, pos // page].long(), pos % page
    first = length - n  # each sequence's first new position: only its block can hold older rows
    fpg = s["table"][torch.arange(len(n), device="cuda"), first // page].long()
    fb = first % page // block
    kv, d = s["k"].shape[2], s["k"].shape[4]
    nb = page // block
    fresh = torch.ones(s["k"].shape[1] * nb, dtype=torch.bool, device="cuda")
    fresh[fpg * nb + fb] = first % block == 0
    at = pg * nb + slot // block
    heads = torch.arange(kv, device="cuda")
    for new, codes, scale in ((s["k_new"], s["k"][0], s["k_scale"][0]), (s["v_new"], s["v"][0], s["v_scale"][0])):
        x = new.float()
        size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
        amax = torch.zeros(fresh.shape[0], kv, device="cuda")
        amax.scatter_reduce_(0, at[:, None].expand(-1, kv), size, "amax")
        was = scale.transpose(1, 2).reshape(-1, kv)
        touched = torch.zeros_like(fresh)
        touched[at] = True
        want = torch.where(amax >= _TINY, amax / 127, 0.0)
        now = torch.where(fresh[:, None], want, torch.maximum(was, want))
        now = torch.where(touched[:, None], now, was)
        # older rows of a block whose scale grew
        ratio = torch.where(now > 0, was / now, 0.0)[fpg * nb + fb]
        old = codes.view(-1, kv, nb, block, d)[fpg, :, fb]
        keep = (torch.arange(block, device="cuda") < (first % block)[:, None])[:, None, :, None]
        codes.view(-1, kv, nb, block, d)[fpg, :, fb] = torch.where(
            keep, torch.round(old.float() * ratio[:, :, None, None]).to(torch.int8), old)
        inv = torch.where(now > 0, 1 / now, 0.0)[at]
        code = torch.round(torch.nan_to_num(x * inv[..., None], nan=0.0)).clamp_(-127, 127).to(torch.int8)
        codes[pg[:, None], heads, slot[:, None]] = code
        scale.copy_(now.view(-1, nb, kv).transpose(1, 2))
    return _plain_rows(s)


def _plain_rows(s):
    """The values that the tokens which the call may have changed stand for."""
    page, block = s["page"], s["block"]
    cu = s["back"].long()
    t = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = s["length"].long()[seq] - cu[seq + 1] + t
    pg, slot = s["table"][seq, pos // page].long(), pos % page
    heads = torch.arange(s["k"].shape[2], device="cuda")
    out = []
    for codes, scale in ((s["k"][0], s["k_scale"][0]), (s["v"][0], s["v_scale"][0])):
        x = codes[pg[:, None], heads, slot[:, None]].float()
        out.append(x * scale[pg[:, None], heads, (slot // block)[:, None]][..., None])
    return {"k": out[0], "v": out[1]}


def _plain_attend(s):
    page = s["page"]
    seq, j, n = _rows_of(s, s["max_n"])
    m, (total, heads, d) = s["length"].shape[0], s["q"].shape
    kv = s["k"].shape[2]
    length = s["length"].long()
    t = s["table"].clamp(min=0).long()

    def dense(codes, scale):  # [m, kv, tokens, d]
        x = codes[0][t].view(m, t.shape[1], kv, page // s["block"], s["block"], d).float()
        x = x * scale[0][t][..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(m, kv, t.shape[1] * page, d)

    q = torch.zeros(m, s["max_n"], heads, d, device="cuda")
    q[seq, j] = s["q"].float()
    q = q.view(m, s["max_n"], kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(m, kv, -1, d)
    score = torch.matmul(q, dense(s["k"], s["k_scale"]).transpose(-1, -2)).mul_(s["scale"])
    p = (length - n)[:, None] + torch.arange(s["max_n"], device="cuda")
    tok = torch.arange(t.shape[1] * page, device="cuda")
    see = (tok <= p[..., None]) & (tok < length[:, None, None])
    if s["window"]:
        see &= (tok > p[..., None] - s["window"]) | (tok < s["sinks"])
    score = score.view(m, kv, heads // kv, s["max_n"], -1).masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    score = score.sub_(top).exp_()
    total_w = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(m, kv, -1, score.shape[-1]), dense(s["v"], s["v_scale"]))
    out = out.view(m, kv, heads // kv, s["max_n"], d) / total_w.clamp(min=1e-30)
    lse = (top + total_w.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(m, s["max_n"], heads, d)[seq, j]
    lse = lse.permute(0, 3, 1, 2).reshape(m, s["max_n"], heads)[seq, j]
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _free_pages(refs):
    """The free pages' ids in ascending order, then the others."""
    return torch.sort((refs > 0).to(torch.int8), stable=True).indices.to(torch.int32)


def _count(refs, table, add):
    refs.scatter_add_(0, table.clamp(min=0).long().flatten(), torch.where(table >= 0, add, 0).int().flatten())


def _buffers(s):
    return {x: s[x] for x in ("table", "length", "refs", "k", "v", "k_scale", "v_scale")}


def _plain_fork(s):
    page, block = s["page"], s["block"]
    child, parent = s["children"].long(), s["parents"].long()
    length = s["length"][parent]
    rows = s["table"][parent]
    used = length % page
    fresh = (used > 0) & (child != parent)
    last = ((length.long() + page - 1) // page - 1).clamp(min=0)
    src = rows.gather(1, last[:, None])[:, 0]
    rank = torch.cumsum(fresh, 0) - fresh.long()
    dst = torch.where(fresh, _free_pages(s["refs"])[rank.clamp(max=s["refs"].shape[0] - 1)], src)
    rows = rows.scatter(1, last[:, None], dst[:, None])
    _count(s["refs"], s["table"][child], -1)
    _count(s["refs"], rows, 1)
    s["table"][child], s["length"][child] = rows, length
    at = fresh.nonzero()[:, 0]
    a, b, u = src[at].long(), dst[at].long(), used[at]
    keep = torch.arange(page, device="cuda") < u[:, None]
    keep_b = torch.arange(page // block, device="cuda") * block < u[:, None]
    for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        codes[:, b] = torch.where(keep[None, :, None, :, None], codes[:, a], codes[:, b])
        scale[:, b] = torch.where(keep_b[None, :, None, :], scale[:, a], scale[:, b])
    return _buffers(s)


def _plain_compact(s):
    for name, was in zip(("table", "refs"), s["was"]):
        s[name].copy_(was)
    live = s["refs"] > 0
    low = torch.arange(live.shape[0], device="cuda") < live.sum()
    src, dst = (live & ~low).nonzero()[:, 0], (~live & low).nonzero()[:, 0]
    move = torch.arange(live.shape[0], device="cuda", dtype=torch.int32)
    move[src] = dst.to(torch.int32)
    s["table"].copy_(torch.where(s["table"] >= 0, move[s["table"].clamp(min=0).long()], s["table"]))
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    for x in ("k", "v", "k_scale", "v_scale"):
        s[x][:, dst] = s[x][:, src]
    return _buffers(s)


def _plain_turnover(s):
    page, seqs = s["page"], s["seqs"].long()
    _count(s["refs"], s["table"][seqs], -1)
    s["table"][seqs] = -1
    s["length"][seqs] = 0
    # pages for the new streams' prompts, the lowest free ones in the streams' order
    need = (s["counts"].long() + page - 1) // page
    at = torch.cumsum(need, 0) - need
    j = torch.arange(s["table"].shape[1], device="cuda")
    rank = (at[:, None] + j).clamp(max=s["refs"].shape[0] - 1)
    rows = torch.where(j < need[:, None], _free_pages(s["refs"])[rank], torch.full_like(s["table"][:1], -1))
    s["table"][seqs] = rows
    s["length"][seqs] = s["counts"]
    _count(s["refs"], rows, 1)
    # whole pages that are before every later query's window and behind the first tokens
    low = (s["length"].long() - s["window"])[:, None]
    out = ((j + 1) * page <= low) & (j * page >= s["sinks"]) & (s["table"] >= 0)
    _count(s["refs"], torch.where(out, s["table"], torch.full_like(s["table"], -1)), -1)
    s["table"].masked_fill_(out, -1)
    return _buffers(s)


# ---- one pass --------------------------------------------------------------------


def _cache(s):
    """The cache object over the state's tensors, made once as a program that serves keeps it."""
    if "cache" not in s:
        from stealcode_b200 import KvCache8

        s["cache"] = KvCache8.wrap(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["length"], s["refs"])
    return s["cache"]


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact,
                "turnover": _plain_turnover}[op](s)
    cache = _cache(s)
    if op == "append":
        cache.append(0, s["k_new"], s["v_new"], cu=s["cu"], n=s["max_n"])
        k, v = cache.rows(0, cu=s["back"], n=s["max_back"], total=s["rows"])
        return {"k": k, "v": v}
    if op == "attend":
        out, lse = cache.attend(0, s["q"], cu=s["cu"], n=s["max_n"], max_len=s["max_len"], window=s["window"],
                                sinks=s["sinks"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "fork":
        cache.fork(s["parents"], s["children"])
    elif op == "compact":
        for name, was in zip(("table", "refs"), s["was"]):
            s[name].copy_(was)
        cache.compact()
    else:
        cache.release(s["seqs"])
        cache.reserve(s["counts"], seqs=s["seqs"])
        cache.slide(s["window"], s["sinks"])
    return _buffers(s)


# ---- work and exact values ---------------------------------------------------------


def _visible(c, length, n):
    """(tokens that some query of the sequence sees, pairs that are seen)."""
    window, sinks = c["window"], c["sinks"]
    if not window:
        return length, n * length - n * (n - 1) // 2
    pairs = 0
    for p in range(length - n, length):
        lo = max(0, p - window + 1)
        pairs += p + 1 - lo + min(sinks, lo)
    lo = max(0, length - n - window + 1)
    return length - lo + min(sinks, lo), pairs


def work(case):
    c = case
    per = 2 * c["kv"] * c["d"]  # bytes of a token's codes
    per_scales = 2 * c["kv"] * 4
    if c["op"] == "append":
        length, n = _lens(c)
        total = sum(n)
        # new rows in, codes out; then the rows that were touched come back as f32
        return {"bytes": total * per * (_SIZE[c["dtype"]] + 1) + sum(_back(c)) * per * (1 + 4), "flops": total * per * 3}
    if c["op"] == "attend":
        length, n = _lens(c)
        seen = [_visible(c, a, b) for a, b in zip(length, n)]
        tokens, pairs = sum(x[0] for x in seen), sum(x[1] for x in seen)
        rows = sum(n) * c["heads"]
        return {"bytes": tokens * per + tokens // c["block"] * per_scales + rows * (c["d"] * 2 * _SIZE[c["dtype"]] + 4),
                "flops": 4 * c["d"] * c["heads"] * pairs}
    if c["op"] == "fork":
        tail = sum(x % c["page"] for x in _spread(c["len_lo"], c["len_hi"], c["m"]))
        copied = tail * (c["beams"] - 1) * c["layers"]  # about one hypothesis in `beams` stays with itself
        table = 2 * 4 * c["m"] * c["beams"] * _pages(c["len_hi"], c["page"])
        return {"bytes": 2 * copied * per + table, "flops": 0}
    owned = [_pages(x, c["page"]) for x in _spread(c["len_lo"], c["len_hi"], c["m"])]
    meta = 4 * (2 * c["m"] * max(owned) + 2 * sum(owned))
    if c["op"] == "compact":
        live = sum(owned[1::2])
        moved = live * (sum(owned) - live) // max(1, sum(owned))
        return {"bytes": 2 * moved * c["page"] * c["layers"] * (per + per_scales / c["block"]) + meta, "flops": 0}
    return {"bytes": meta, "flops": 0}


def _exact_append(s):
    """The changed tokens' stored values of each sequence, in 64 bits."""
    c, page, block = s["case"], s["page"], s["block"]
    out = {"k": [], "v": []}
    at = 0
    for i, (end, new) in enumerate(zip(*_lens(c))):
        start = end - new
        lo = start // block * block
        pos = torch.arange(lo, end, device="cuda")
        pages = s["table"][i].long()[pos // page]
        group = pos // block - lo // block
        for codes, scales, rows, name in ((s["k"], s["k_scale"], s["k_new"], "k"), (s["v"], s["v_scale"], s["v_new"], "v")):
            was = scales[0, pages, :, pos % page // block].double()
            old = codes[0, pages, :, pos % page].double() * was[..., None]
            x = rows[at:at + new].double()
            amax = torch.zeros(int(group[-1]) + 1, c["kv"], dtype=torch.float64, device="cuda")
            amax.index_reduce_(0, group[start - lo:], x.abs().amax(-1), "amax")
            step = amax / 127
            if start > lo:
                step[0] = torch.maximum(step[0], was[0])
            step = step[group][..., None]
            out[name].append(torch.round(torch.cat([old[:start - lo], x]) / step) * step)
        at += new
    return {x: torch.cat(v) for x, v in out.items()}


def _exact_attend(s):
    """Each sequence and key head by itself, over the tokens that can be seen, in 64 bits."""
    c, page, block = s["case"], s["page"], s["block"]
    length, n = _lens(c)
    group = c["heads"] // c["kv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for i, (end, new) in enumerate(zip(length, n)):
        tok = torch.arange(end, device="cuda")
        if c["window"]:
            tok = tok[(tok > end - new - c["window"]) | (tok < c["sinks"])]
        pages = s["table"][i].long()[tok // page]
        p = torch.arange(end - new, end, device="cuda")[:, None]
        hide = tok[None] > p
        if c["window"]:
            hide |= (tok[None] <= p - c["window"]) & (tok[None] >= c["sinks"])
        for h in range(c["kv"]):
            k, v = (codes[0, pages, h, tok % page].double() * scale[0, pages, h, tok % page // block].double()[:, None]
                    for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
            q = s["q"][at:at + new, h * group:(h + 1) * group].double()
            w = torch.einsum("ngd,td->gnt", q, k) * s["scale"]
            w.masked_fill_(hide, -math.inf)
            z = torch.logsumexp(w, -1)
            out[at:at + new, h * group:(h + 1) * group] = torch.einsum("gnt,td->ngd", torch.exp(w - z[..., None]), v)
            lse[at:at + new, h * group:(h + 1) * group] = z.T
        at += new
    return {"out": out, "lse": lse}


def exact(case, seed):
    """The outputs in 64 bits; the page operations move whole numbers and have no such values."""
    if case["op"] not in ("append", "attend"):
        return None
    s = prepare(case, seed)
    return (_exact_append if case["op"] == "append" else _exact_attend)(s)
