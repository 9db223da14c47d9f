"""The attention operators of a language or image-text model as a serving program calls them:
rotary positions with several axes, appending rotated keys and values to a paged cache, attention
over that cache, and attention over ragged prompts with a sliding window and first tokens that
stay visible.  listed() gives the calls that are timed, draw() more of the same ranges; run() takes
a call's plain form in elementary torch operations, or the framework's entry points where `own`
is set; exact() the same results in 64 bits.

Layouts: a token's rows are [tokens][heads][dim].  A cache page holds `page` tokens of every head;
with E = 16 bytes' worth of elements (16 codes of 8 bits, 8 values of 16 bits) keys are stored as
[pages][heads][page / 4][dim / E][4][E] and values as [pages][heads][page / E][dim][E].  8-bit pages
hold e4m3 codes with one fp32 scale for each page and head, a power of two.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LOWEST = 2.0 ** -32  # smallest scale of an 8-bit page


# ------------------------------------------------------------------------------ the cases
def rope(name=None, **kw):
    c = {"kind": "rope", "type": "bf16", "tokens": 1, "heads": 32, "dim": 128, "rot": 128, "axes": 1, "adjacent": False,
         "dealt": False, "per_axis": False, "packed": False}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def append(name=None, **kw):
    c = {"kind": "append", "type": "bf16", "bits": 8, "batch": 1, "heads": 8, "dim": 128, "rot": 128, "axes": 1,
         "adjacent": False, "dealt": False, "per_axis": False, "page": 16, "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 0,
         "pad": 0}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def paged(name=None, **kw):
    c = {"kind": "paged", "type": "bf16", "bits": 8, "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "new_lo": 1, "new_hi": 1, "len_lo": 1, "len_hi": 1, "window": 0, "sinks": 0, "pad": 0}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def attention(name=None, **kw):
    c = {"kind": "attention", "type": "bf16", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 64, "len_lo": 1, "len_hi": 1,
         "causal": True, "window": 0, "sinks": 0}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one generated token's queries and keys in a decoding step: the smallest call, latency counts
        rope("rope_one_token", tokens=1, heads=40),
        # patches of four 640-pixel images at 16 pixels a patch in an image encoder: two axes, each
        # with a frequency ladder of its own, heads of 80 channels cut from packed q, k, v rows
        rope("rope_images_2_axes", type="f16", tokens=6400, heads=32, dim=80, rot=80, axes=2, per_axis=True, packed=True),
        # a long video prompt of a language model: time, height and width share the frequencies
        rope("rope_video_3_axes", tokens=32768, heads=40, axes=3, dealt=True),
        # one generated token of each of 64 sequences into an 8-bit cache, some rows of padding
        append("append_decode", type="f16", batch=60, old_lo=1, old_hi=9000, pad=4),
        # ragged prompts, some behind tokens that are cached already, into an 8-bit cache
        append("append_prompts", batch=9, heads=8, axes=3, page=64, new_lo=257, new_hi=4811, old_lo=0, old_hi=300),
        # chunks of prompts into a cache of the model's own type; half of each head's channels turn
        append("append_16bit_chunks", bits=16, batch=12, heads=4, dim=256, rot=64, adjacent=True, page=32, new_lo=33,
               new_hi=1024, old_lo=5, old_hi=4000),
        # one sequence that generates a token, 5000 tokens behind it: latency counts
        paged("paged_one_sequence", batch=1, len_lo=5003, len_hi=5003),
        # a full decoding batch of ragged long sequences: the throughput step
        paged("paged_long_batch", type="f16", batch=64, len_lo=900, len_hi=16001, page=32, pad=8),
        # five drafted tokens of each sequence verified at once, a window of 1024 and 4 first tokens
        paged("paged_window_draft", batch=24, heads=32, kv_heads=4, new_lo=5, new_hi=5, len_lo=600, len_hi=20000, window=1024,
              sinks=4, page=64),
        # one long prompt, every earlier token visible: the largest call
        attention("attention_prompt", heads=16, kv_heads=4, dim=128, len_lo=16384, len_hi=16384),
        # ragged prompts with a sliding window and a few first tokens
        attention("attention_window_prompts", batch=5, heads=16, kv_heads=8, dim=128, len_lo=701, len_hi=6007, window=1024,
                  sinks=16),
        # images of up to 20x20 patches in an encoder, every patch visible to every other
        attention("attention_images", type="f16", batch=64, heads=16, kv_heads=16, dim=72, len_lo=289, len_hi=400,
                  causal=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "paged", "attention"])
    t = rng.choice(["f16", "bf16"])
    if kind == "rope":
        while True:
            dim = rng.choice([64, 72, 80, 96, 128, 128, 256])
            rot = dim if rng.random() < 0.7 else max(16, dim // 2 // 8 * 8)
            axes = rng.choice([1, 1, 2, 3])
            c = rope(type=t, tokens=_log(rng, 1, 32768), heads=rng.choice([1, 5, 8, 16, 28, 40]), dim=dim, rot=rot, axes=axes,
                     adjacent=rng.random() < 0.3, dealt=axes > 1 and rng.random() < 0.5, packed=rng.random() < 0.4)
            c["per_axis"] = axes > 1 and not c["dealt"] and rng.random() < 0.5
            if c["tokens"] * c["heads"] * dim <= 32768 * 40 * 128:
                return c
    if kind == "append":
        while True:
            dim = rng.choice([64, 80, 96, 128, 128, 256])
            rot = dim if rng.random() < 0.7 else max(16, dim // 2 // 8 * 8)
            axes = rng.choice([1, 1, 2, 3])
            hi = _log(rng, 1, 4811)
            old = _log(rng, 1, 9000)
            c = append(type=t, bits=rng.choice([8, 8, 16]), batch=_log(rng, 1, 128), heads=rng.choice([1, 2, 4, 8]), dim=dim,
                       rot=rot, axes=axes, adjacent=rng.random() < 0.3, dealt=axes > 1 and rng.random() < 0.5,
                       page=rng.choice([16, 32, 64, 128]), new_lo=max(0, hi // 3), new_hi=hi, old_lo=old // 5, old_hi=old,
                       pad=rng.choice([0, 0, 3, 17]))
            if sum(_appended(c)[0]) * c["heads"] * dim <= 9 * 4811 * 8 * 128 and sum(_appended(c)[1]) <= 300000:
                return c
    if kind == "paged":
        while True:
            hi = _log(rng, 1, 20000)
            new = rng.choice([1, 1, 1, 2, 5, 8, _log(rng, 1, 300)])
            kv = rng.choice([1, 2, 4, 8])
            c = paged(type=t, bits=rng.choice([8, 8, 16]), batch=_log(rng, 1, 96), heads=kv * rng.choice([1, 3, 4, 7, 8]),
                      kv_heads=kv, dim=rng.choice([64, 80, 96, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]),
                      new_lo=max(1, new // 2), new_hi=new, len_lo=max(new, hi // 4), len_hi=max(new, hi), pad=rng.choice([0, 0, 2, 9]))
            if rng.random() < 0.4:
                c.update(window=_log(rng, 1, 2048), sinks=rng.choice([0, 1, 4, 64]))
            if c["batch"] * c["len_hi"] * kv * c["dim"] * c["bits"] <= 64 * 16001 * 8 * 128 * 8 and \
                    c["batch"] * new * c["heads"] * c["len_hi"] <= 1 << 30:
                return c
    while True:
        hi = _log(rng, 1, 16384)
        kv = rng.choice([1, 2, 4, 8, 16])
        c = attention(type=t, batch=_log(rng, 1, 64), heads=kv * rng.choice([1, 1, 2, 4]), kv_heads=kv,
                      dim=rng.choice([32, 64, 72, 80, 96, 128, 128, 256]), len_lo=max(1, hi // 3), len_hi=hi,
                      causal=rng.random() < 0.6)
        if rng.random() < 0.5:
            c.update(window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 16, 100]))
        if c["batch"] * c["heads"] * hi * hi <= 16 * 16384 * 16384 and c["batch"] * c["heads"] * hi * hi * c["dim"] <= 16 * 16384 ** 2 * 128:
            return c


# ------------------------------------------------------------------------------ sizes
def _spread(n, lo, hi, shift=0.0):
    """n lengths between lo and hi, the first of them hi where shift is 0: fixed, and in no order."""
    return [lo + int(round((hi - lo) * (1.0 - (b * 0.6180339887498949 + shift) % 1.0))) for b in range(n)]


def _appended(c):
    """(new, old) tokens of each sequence."""
    return _spread(c["batch"], c["new_lo"], c["new_hi"]), _spread(c["batch"], c["old_lo"], c["old_hi"], 0.37)


def _cached(c):
    """(new, all) tokens of each sequence."""
    new, full = _spread(c["batch"], c["new_lo"], c["new_hi"]), _spread(c["batch"], c["len_lo"], c["len_hi"])
    return new, [max(n, f) for n, f in zip(new, full)]


def _sections(c):
    """Frequencies of each axis: equal parts, what is left over to the first."""
    half, axes = c["rot"] // 2, c["axes"]
    part = half // axes
    return [half - part * (axes - 1)] + [part] * (axes - 1)


def _axes(c):
    """The axis of each frequency: the axes' sections one after the other, or dealt in turn."""
    half, axes, sections = c["rot"] // 2, c["axes"], _sections(c)
    if not c["dealt"]:
        return [a for a in range(axes) for _ in range(sections[a])]
    return [f % axes if f % axes and f // axes < sections[f % axes] else 0 for f in range(half)]


def _ladder(c):
    """Rotation in radians of one position step, for each frequency."""
    half = c["rot"] // 2
    if c["per_axis"]:  # each axis has a ladder of its own
        return [10000.0 ** (-f / s) for s in _sections(c) for f in range(s)]
    return [1000000.0 ** (-f / half) for f in range(half)]


def _visible(nq, nk, causal, window, sinks):
    """Query and key pairs of one sequence whose last query stands at its last key."""
    i = np.arange(nk - nq, nk, dtype=np.int64)
    hi = np.minimum(i, nk - 1) if causal else np.full(nq, nk - 1, dtype=np.int64)
    lo = np.zeros(nq, dtype=np.int64)
    if window:
        lo = np.maximum(0, i - window + 1)
        hi = np.minimum(hi, i + window - 1)
    lo = np.minimum(lo, nk)
    return int(np.maximum(0, hi - lo + 1).sum() + (np.minimum(lo, sinks).sum() if window else 0))


def _reached(nq, nk, window, sinks):
    """Keys of one sequence that some query of the last nq sees."""
    lo = max(0, nk - nq - window + 1) if window else 0
    return nk - lo + min(lo, sinks)


def work(case):
    c = case
    if c["kind"] == "rope":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 4 * n + 4 * c["tokens"] * c["axes"] + 2 * c["rot"], "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    if c["kind"] == "append":
        new, old = _appended(c)
        n = sum(new) * c["heads"] * c["dim"]
        pages = sum(-(-(o + k) // c["page"]) - o // c["page"] for k, o in zip(new, old) if k)
        scales = 2 * 4 * pages * c["heads"] if c["bits"] == 8 else 0
        return {"bytes": 2 * n * 2 + 2 * n * c["bits"] // 8 + scales + 4 * sum(new) * c["axes"] + 4 * pages,
                "flops": 3 * sum(new) * c["heads"] * c["rot"] + (4 * n if c["bits"] == 8 else 0)}
    if c["kind"] == "paged":
        new, full = _cached(c)
        keys = sum(_reached(n, f, c["window"], c["sinks"]) for n, f in zip(new, full))
        pairs = sum(_visible(n, f, True, c["window"], c["sinks"]) for n, f in zip(new, full))
        scale = 8.0 / c["page"] if c["bits"] == 8 else 0
        return {"bytes": keys * c["kv_heads"] * (2 * c["dim"] * c["bits"] / 8 + scale) + 4 * keys / c["page"] +
                4 * sum(new) * c["heads"] * c["dim"], "flops": 4 * pairs * c["heads"] * c["dim"]}
    full = _spread(c["batch"], c["len_lo"], c["len_hi"])
    pairs = sum(_visible(n, n, c["causal"], c["window"], c["sinks"]) for n in full)
    return {"bytes": 2 * sum(full) * c["dim"] * (2 * c["heads"] + 2 * c["kv_heads"]), "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------------------ inputs
def _positions(c, starts, counts, gen):
    """int32 [axes][tokens]: text counts on; images and video have a place on each axis."""
    dev = gen.device
    total = sum(counts)
    if c["axes"] == 1:
        first = torch.tensor([s - b for s, b in zip(starts, np.cumsum([0] + counts[:-1]).tolist())], device=dev)
        at = torch.repeat_interleave(first, torch.tensor(counts, device=dev)) + torch.arange(total, device=dev)
        return at.to(torch.int32).reshape(1, total).contiguous()
    t = torch.arange(total, device=dev)
    w, h = 40, 25
    rows = [t // (w * h), t // w % h, t % w][3 - c["axes"]:]
    base = int(torch.randint(0, 5000, (1,), generator=gen, device=dev))
    return (torch.stack(rows) + base).to(torch.int32).contiguous()


def _scale8(amax):
    """The smallest power of two s with amax <= 448 s, at least LOWEST."""
    m, e = torch.frexp(amax / 448.0)
    return torch.ldexp(torch.ones_like(amax), e - (m == 0.5).to(e.dtype)).clamp(min=LOWEST)


def _each(c):
    return 16 if c["bits"] == 8 else 8  # elements of 16 bytes


def _pack_keys(x, c):  # [pages][heads][page][dim] -> the stored order
    p, h, n, d = x.shape
    e = _each(c)
    return x.reshape(p, h, n // 4, 4, d // e, e).permute(0, 1, 2, 4, 3, 5).contiguous()


def _pack_values(x, c):
    p, h, n, d = x.shape
    e = _each(c)
    return x.reshape(p, h, n // e, e, d).permute(0, 1, 2, 4, 3).contiguous()


def _cache(c, pages, gen):
    """Pages of normal keys and values, each page and head with a magnitude of its own."""
    t, kv = TYPES[c["type"]], c["kv_heads"] if c["kind"] == "paged" else c["heads"]
    got = []
    for pack in (_pack_keys, _pack_values):
        x = torch.randn((pages, kv, c["page"], c["dim"]), generator=gen, device=gen.device)
        x *= torch.exp2(0.5 * torch.randn((pages, kv, 1, 1), generator=gen, device=gen.device))
        if c["bits"] == 16:
            got += [pack(x.to(t), c), None]
        else:
            s = _scale8(x.abs().amax((2, 3)))
            got += [pack((x / s[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8), c).view(torch.float8_e4m3fn), s]
    return got


def _table(c, full, gen):
    """(page of each sequence and place, pages in all): pages in no order, unused places -1."""
    used = [-(-n // c["page"]) for n in full]
    pages, width = sum(used) + 3, max(max(used), 1) + 1
    order = torch.randperm(pages, generator=gen, device=gen.device).to(torch.int32)
    first = torch.tensor(np.cumsum([0] + used[:-1]), device=gen.device)
    at = torch.arange(width, device=gen.device)
    live = at[None, :] < torch.tensor(used, device=gen.device)[:, None]
    table = torch.where(live, order[(first[:, None] + at).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=gen.device))
    return table.to(torch.int32).contiguous(), pages, width


def _ends(counts, dev):
    return torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=dev)


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    t = TYPES[c["type"]]
    rand = lambda *shape: torch.randn(shape, generator=gen, device=dev).to(t)  # noqa: E731
    s = {"case": c}
    if c["kind"] in ("rope", "append"):
        s["freq"] = torch.tensor(_ladder(c), dtype=torch.float32, device=dev)
    if c["kind"] == "rope":
        wide = (c["heads"] + ((c["heads"] + 1) // 2 if c["packed"] else 0)) * c["dim"]  # q and k of packed q, k, v rows
        s["rows"] = rand(c["tokens"], wide)
        s["x"] = s["rows"][:, :c["heads"] * c["dim"]].unflatten(1, (c["heads"], c["dim"]))
        start = int(torch.randint(0, 900000, (1,), generator=gen, device=dev))
        s["pos"] = _positions(c, [start], [c["tokens"]], gen)
        s["y"] = torch.zeros((c["tokens"], c["heads"], c["dim"]), dtype=t, device=dev)
    elif c["kind"] == "append":
        new, old = _appended(c)
        full = [a + b for a, b in zip(new, old)]
        rows = sum(new) + c["pad"]
        s["k"], s["v"] = rand(rows, c["heads"], c["dim"]), rand(rows, c["heads"], c["dim"])
        pos = _positions(c, old, new, gen)
        s["pos"] = torch.cat([pos, torch.zeros((c["axes"], c["pad"]), dtype=torch.int32, device=dev)], 1).contiguous()
        s["cu"], s["lens"] = _ends(new, dev), torch.tensor(full, dtype=torch.int32, device=dev)
        s["table"], s["pages"], s["width"] = _table(c, full, gen)
        s["kc"], s["ks"], s["vc"], s["vs"] = _cache(c, s["pages"] + 1, gen)  # one page that belongs to no sequence
        s["rows"] = rows
    elif c["kind"] == "paged":
        new, full = _cached(c)
        rows = sum(new) + c["pad"]
        s["q"] = rand(rows, c["heads"], c["dim"])
        s["cu"], s["lens"] = _ends(new, dev), torch.tensor(full, dtype=torch.int32, device=dev)
        s["table"], s["pages"], s["width"] = _table(c, full, gen)
        s["kc"], s["ks"], s["vc"], s["vs"] = _cache(c, s["pages"], gen)
        s["o"] = torch.zeros((rows, c["heads"], c["dim"]), dtype=t, device=dev)
        s["rows"], s["max_new"], s["max_len"] = rows, max(new), max(full)
    else:
        full = _spread(c["batch"], c["len_lo"], c["len_hi"])
        n = sum(full)
        s["q"], s["k"], s["v"] = rand(n, c["heads"], c["dim"]), rand(n, c["kv_heads"], c["dim"]), rand(n, c["kv_heads"], c["dim"])
        s["cu"] = _ends(full, dev)
        s["o"] = torch.zeros((n, c["heads"], c["dim"]), dtype=t, device=dev)
        s["rows"], s["max_len"] = n, max(full)
    return s


# ------------------------------------------------------------------------------ the plain forms
def _turned(x, pos, freq, c):
    """x [tokens][heads][dim] with its first `rot` channels rotated, in 32 bits; angles in 64."""
    axis = torch.tensor(_axes(c), device=x.device)
    angle = pos.double()[axis].t() * freq.double()  # [tokens][rot / 2]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = x.float()
    rot, half = c["rot"], c["rot"] // 2
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["adjacent"] else (x[..., :half], x[..., half:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if c["adjacent"] else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _places(cu, rows):
    """(sequence, index among its new rows) of each row; rows behind the last sequence get it too."""
    at = torch.arange(rows, device=cu.device, dtype=torch.int32)
    b = (torch.searchsorted(cu, at, right=True) - 1).clamp(0, cu.numel() - 2)
    return b, at - cu[b]


def _plain_append(s):
    c = s["case"]
    n = sum(_appended(c)[0])
    k, v = _turned(s["k"][:n], s["pos"][:, :n], s["freq"], c), s["v"][:n].float()
    b, i = _places(s["cu"], n)
    new = s["cu"][1:] - s["cu"][:-1]
    old = s["lens"] - new
    at = old[b] + i
    page = s["table"][b, at // c["page"]].long()
    slot = (at % c["page"]).long()
    e = _each(c)
    for x, buf, scales, keys in ((k, s["kc"], s["ks"], True), (v, s["vc"], s["vs"], False)):
        if scales is None:
            store, codes = buf, x.to(buf.dtype)
        else:
            amax = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(2), "amax")
            need = torch.zeros_like(scales, dtype=torch.bool).index_fill_(0, page, True)
            # the first page a sequence writes may hold older tokens, whose codes follow the scale;
            # the sequences without one share the last page, which no sequence has
            part = (new > 0) & (old % c["page"] > 0)
            first = torch.where(part, s["table"].gather(1, (old // c["page"])[:, None].long())[:, 0], s["pages"]).long()
            held = torch.zeros(scales.shape[0], dtype=torch.bool, device=x.device).index_fill_(0, first, True)[:, None]
            scale = torch.where(need, torch.maximum(_scale8(amax), torch.where(held, scales, 0.0)), scales)
            store = buf.view(torch.uint8)
            moved = buf[first].float() * (scales[first] / scale[first]).reshape(first.shape + scale.shape[1:] + (1,) * (buf.dim() - 2))
            store.index_copy_(0, first, moved.to(buf.dtype).view(torch.uint8))
            codes = (x / scale[page][..., None]).to(buf.dtype).view(torch.uint8)
            scales.copy_(scale)
        if keys:
            store[page, :, slot // 4, :, slot % 4] = codes.unflatten(2, (-1, e))
        else:
            store[page, :, slot // e, :, slot % e] = codes
    return _pages(s)


def _pages(s):
    return [x[:s["pages"]] for x in (s["kc"], s["ks"], s["vc"], s["vs"]) if x is not None]


def _plain_attend(q, k, v, at, full, causal, window, sinks):
    """q [B][heads][n][dim], k and v [B][kv][keys][dim] in 32 bits; query places `at` [B][n], `full`
    keys of each sequence.  A row that sees nothing is zero."""
    b, heads, n, d = q.shape
    kv, keys = k.shape[1], k.shape[2]
    j = torch.arange(keys, device=q.device)
    i = at[:, :, None]
    seen = (j < full[:, None, None]) & ((j <= i) if causal else (i >= -keys))
    if window:
        seen = seen & (((i - j).abs() < window) | (j < sinks))
    seen = seen[:, None, None]
    x = torch.matmul(q.reshape(b, kv, heads // kv * n, d), k.transpose(2, 3)).reshape(b, kv, heads // kv, n, keys)
    x = x.mul_(1.0 / math.sqrt(d)).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(b, kv, heads // kv * n, keys), v).reshape(b, kv, heads // kv, n, d)
    return (o / torch.where(total == 0, 1.0, total)).reshape(b, heads, n, d)


def _padded(x, cu, n):
    """[rows][heads][dim] -> [batch][heads][n][dim] in 32 bits, zeros behind a sequence's rows."""
    at = cu[:-1, None] + torch.arange(n, device=x.device)
    live = at < cu[1:, None]
    got = x[at.clamp(max=x.shape[0] - 1).long()].float() * live[:, :, None, None]
    return got.permute(0, 2, 1, 3)


def _plain_paged(s):
    c = s["case"]
    n, kv = s["max_new"], c["kv_heads"]
    pages = s["table"].clamp(min=0).long()
    k, v = s["kc"], s["vc"]
    if c["bits"] == 8:
        k = k.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["ks"][pages][..., None, None, None, None]
        v = v.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["vs"][pages][..., None, None, None]
    else:
        k, v = k[pages].float(), v[pages].float()
    b, w = pages.shape
    k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(b, kv, w * c["page"], c["dim"])
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(b, kv, w * c["page"], c["dim"])
    at = (s["lens"] - (s["cu"][1:] - s["cu"][:-1]))[:, None] + torch.arange(n, device=k.device)
    live = torch.arange(w * c["page"], device=k.device) < s["lens"][:, None]
    o = _plain_attend(_padded(s["q"], s["cu"], n), k * live[:, None, :, None], v * live[:, None, :, None], at, s["lens"], True,
                      c["window"], c["sinks"])
    seq, i = _places(s["cu"], s["rows"])
    rows = o[seq, :, i.clamp(max=n - 1)].to(s["q"].dtype)
    return torch.where((torch.arange(s["rows"], device=k.device) < s["cu"][-1])[:, None, None], rows, s["o"])


def _plain_attention(s):
    c = s["case"]
    n, cu = s["max_len"], s["cu"]
    at = torch.arange(n, device=cu.device).expand(c["batch"], n)
    o = _plain_attend(_padded(s["q"], cu, n), _padded(s["k"], cu, n), _padded(s["v"], cu, n), at, cu[1:] - cu[:-1], c["causal"],
                      c["window"], c["sinks"])
    seq, i = _places(cu, s["rows"])
    return o[seq, :, i].to(s["q"].dtype)


# ------------------------------------------------------------------------------ the framework's calls
def _turning(c):
    return {"sections": _sections(c), "rot": c["rot"], "adjacent": c["adjacent"], "dealt": c["dealt"]}


def _plan(s, ops):
    """Descriptors and the workspace that a program makes once for its shapes."""
    c = s["case"]
    t = ops.F16 if c["type"] == "f16" else ops.BF16
    strides = lambda x: (x.stride(0), x.stride(1))  # noqa: E731
    if c["kind"] == "rope":
        return ops.rope_desc(t, c["heads"], c["dim"], x=strides(s["x"]), y=strides(s["y"]), pos_axis=s["pos"].stride(0), **_turning(c))
    if c["kind"] == "append":
        cache = ops.cache_desc(t, c["bits"], c["heads"], c["dim"], c["page"], s["pages"], s["width"])
        return ops.append_desc(cache, k=strides(s["k"]), v=strides(s["v"]), pos_axis=s["pos"].stride(0), **_turning(c))
    if c["kind"] == "paged":
        cache = ops.cache_desc(t, c["bits"], c["kv_heads"], c["dim"], c["page"], s["pages"], s["width"])
        d = ops.paged_attention_desc(cache, c["heads"], 1.0 / math.sqrt(c["dim"]), window=c["window"], sinks=c["sinks"],
                                     q=strides(s["q"]), o=strides(s["o"]), max_new=s["max_new"], max_len=s["max_len"])
        need = ops.paged_attention_workspace(d, c["batch"], s["rows"])
        return d, torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda"), need
    return ops.attention_desc(t, c["heads"], c["kv_heads"], c["dim"], 1.0 / math.sqrt(c["dim"]), causal=c["causal"],
                              window=c["window"], sinks=c["sinks"], q=strides(s["q"]), k=strides(s["k"]), v=strides(s["v"]),
                              o=strides(s["o"]), max_q=s["max_len"])


def _own_run(s):
    from infvino_amd import ops
    c = s["case"]
    if "plan" not in s:
        s["plan"] = _plan(s, ops)
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    if c["kind"] == "rope":
        ops.rope(s["plan"], at(s["x"]), at(s["pos"]), at(s["freq"]), at(s["y"]), c["tokens"], stream)
        return s["y"]
    if c["kind"] == "append":
        ops.kv_append(s["plan"], at(s["k"]), at(s["v"]), at(s["pos"]), at(s["freq"]), at(s["cu"]), at(s["lens"]), at(s["table"]),
                      at(s["kc"]), at(s["vc"]), at(s["ks"]), at(s["vs"]), c["batch"], s["rows"], stream)
        return _pages(s)
    if c["kind"] == "paged":
        d, space, need = s["plan"]
        ops.paged_attention(d, at(s["q"]), at(s["kc"]), at(s["vc"]), at(s["ks"]), at(s["vs"]), at(s["cu"]), at(s["lens"]),
                            at(s["table"]), at(s["o"]), c["batch"], s["rows"], at(space), need, stream)
        return s["o"]
    ops.attention(s["plan"], at(s["q"]), at(s["k"]), at(s["v"]), at(s["cu"]), at(s["cu"]), at(s["o"]), c["batch"], s["rows"],
                  s["rows"], stream)
    return s["o"]


def run(state):
    if own:
        return _own_run(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        c = state["case"]
        return _turned(state["x"], state["pos"], state["freq"], c).to(state["x"].dtype)
    return {"append": _plain_append, "paged": _plain_paged, "attention": _plain_attention}[kind](state)


# ------------------------------------------------------------------------------ in 64 bits
def _exact_turned(x, pos, freq, c):
    """Channel by channel as a complex product: a pair (a, b) is a + ib, turned by e^(i angle)."""
    y = x.double().clone()
    half = c["rot"] // 2
    for f, a in enumerate(_axes(c)):
        m, n = (2 * f, 2 * f + 1) if c["adjacent"] else (f, f + half)
        angle = pos[a, :x.shape[0]].double() * float(freq[f])
        z = torch.complex(x[..., m].double(), x[..., n].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[..., m], y[..., n] = z.real, z.imag
    return y


def _e4m3(x):
    """x rounded to the nearest e4m3 value, ties to even: three bits behind the leading one, the
    last place no smaller than 2^-9."""
    place = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3
    step = torch.exp2(place)
    return torch.round(x / step) * step


def _exact_append(s):
    c = s["case"]
    new, old = _appended(c)
    k, v = _exact_turned(s["k"][:sum(new)], s["pos"], s["freq"], c), s["v"][:sum(new)].double()
    p, h, n, d = s["pages"], c["heads"], c["page"], c["dim"]
    kc = s["kc"][:p].double().permute(0, 1, 2, 4, 3, 5).reshape(p, h, n, d)
    vc = s["vc"][:p].double().permute(0, 1, 2, 4, 3).reshape(p, h, n, d)
    table = s["table"].tolist()
    ks, vs = (None, None) if c["bits"] == 16 else (s["ks"][:p].double(), s["vs"][:p].double())
    row = 0
    for b in range(c["batch"]):
        at, end = old[b], old[b] + new[b]
        while at < end:
            page, lo = table[b][at // n], at % n
            hi = min(n, lo + end - at)
            for x, buf, scales in ((k, kc, ks), (v, vc, vs)):
                part = x[row:row + hi - lo].transpose(0, 1)
                if scales is None:
                    buf[page, :, lo:hi] = part
                    continue
                need = part.abs().amax((1, 2)) / 448.0
                scale = torch.exp2(torch.ceil(torch.log2(need.clamp(min=LOWEST))))
                if lo:
                    scale = torch.maximum(scale, scales[page])
                    buf[page] = _e4m3(buf[page] * (scales[page] / scale)[:, None, None])
                scales[page] = scale
                buf[page, :, lo:hi] = _e4m3(part / scale[:, None, None])
            row, at = row + hi - lo, at + hi - lo
    e = _each(c)
    kc = kc.reshape(p, h, n // 4, 4, d // e, e).permute(0, 1, 2, 4, 3, 5)
    vc = vc.reshape(p, h, n // e, e, d).permute(0, 1, 2, 4, 3)
    return [kc, vc] if ks is None else [kc, ks, vc, vs]


def _exact_rows(q, k, v, first, c, causal):
    """One sequence and one key head: q [group][n][dim] whose first row stands at `first`."""
    n, keys = q.shape[1], k.shape[0]
    out = torch.empty_like(q)
    block = max(1, (1 << 27) // max(1, keys * q.shape[0]))
    for r in range(0, n, block):
        i = first + torch.arange(r, min(n, r + block), device=q.device)[:, None]
        j = torch.arange(keys, device=q.device)[None]
        hide = (j > i) if causal else torch.zeros_like(j > i)
        if c["window"]:
            hide = hide | (((j - i).abs() >= c["window"]) & (j >= c["sinks"]))
        x = (q[:, r:r + block] @ k.t() / math.sqrt(c["dim"])).masked_fill(hide, -math.inf)
        p = torch.softmax(x, -1).masked_fill(hide, 0.0)
        out[:, r:r + block] = p @ v
    return torch.nan_to_num(out)


def _exact_paged(s):
    c = s["case"]
    new, full = _cached(c)
    if sum(n * f for n, f in zip(new, full)) * c["heads"] * c["dim"] > 1 << 40:
        return None
    o = s["o"].double().clone()
    table, row, group = s["table"].tolist(), 0, c["heads"] // c["kv_heads"]
    for b in range(c["batch"]):
        ids = table[b][:-(-full[b] // c["page"])]
        k, v = s["kc"][ids].double(), s["vc"][ids].double()
        if c["bits"] == 8:
            k, v = k * s["ks"][ids].double()[..., None, None, None, None], v * s["vs"][ids].double()[..., None, None, None]
        k = k.permute(1, 0, 2, 4, 3, 5).reshape(c["kv_heads"], -1, c["dim"])[:, :full[b]]
        v = v.permute(1, 0, 2, 4, 3).reshape(c["kv_heads"], -1, c["dim"])[:, :full[b]]
        for h in range(c["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            q = s["q"][row:row + new[b], mine].double().transpose(0, 1)
            o[row:row + new[b], mine] = _exact_rows(q, k[h], v[h], full[b] - new[b], c, True).transpose(0, 1)
        row += new[b]
    return o


def _exact_attention(s):
    c = s["case"]
    o, row, group = s["o"].double().clone(), 0, c["heads"] // c["kv_heads"]
    for n in _spread(c["batch"], c["len_lo"], c["len_hi"]):
        rows = slice(row, row + n)
        for h in range(c["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            q = s["q"][rows, mine].double().transpose(0, 1)
            o[rows, mine] = _exact_rows(q, s["k"][rows, h].double(), s["v"][rows, h].double(), 0, c, c["causal"]).transpose(0, 1)
        row += n
    return o


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_turned(s["x"], s["pos"], s["freq"], case)
    return {"append": _exact_append, "paged": _exact_paged, "attention": _exact_attention}[case["kind"]](s)
