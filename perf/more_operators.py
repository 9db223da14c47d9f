"""The operators of a program that answers one prompt many times: attention over a paged cache
whose first pages several sequences share, linear attention with a decay for each head (prompts in chunks, single
tokens by recurrence), and the choice of the next token from logits and given random numbers.
listed() gives the calls that are timed, draw() more of the same ranges; run() takes a call's plain
form in elementary torch operations, or the framework's entry points where `own` is set; exact()
the same results in 64 bits.

Layouts: a token's rows are [tokens][heads][dim].  A cache page holds `page` tokens of every head; with E = 16 bytes'
worth of elements keys are stored as [pages][heads][page / 4][dim / E][4][E] and values as
[pages][heads][page / E][dim][E].  8-bit pages hold e4m3 codes with one fp32 scale, a power of two, for each page
and head.  States of the linear attention are fp32 [slots][heads][key_dim][dim].
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 128  # tokens of a step of the plain linear attention


# ------------------------------------------------------------------------------ the cases
def prefix(name=None, **kw):
    c = {"kind": "prefix", "type": "bf16", "bits": 8, "batch": 1, "groups": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "new_lo": 1, "new_hi": 1, "shared_lo": 0, "shared_hi": 0, "own_lo": 1, "own_hi": 1, "pad": 0}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def linear(name=None, **kw):
    c = {"kind": "linear", "type": "bf16", "batch": 1, "heads": 32, "key_heads": 32, "key_dim": 128, "dim": 128, "new_lo": 1,
         "new_hi": 1, "each": True, "fresh": False, "pad": 0}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def sample(name=None, **kw):
    c = {"kind": "sample", "type": "f32", "rows": 1, "vocab": 131072, "top_k": True, "top_p": True, "min_p": False, "greedy": False,
         "masked": False, "pad": 0}
    c.update(kw)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # four answers to one prompt of 2000 tokens, one token each: latency counts
        prefix("prefix_four_answers", batch=4, shared_lo=2000, shared_hi=2000, own_lo=1, own_hi=201),
        # a decoding batch behind a common instruction of 8192 tokens
        prefix("prefix_batch", type="f16", batch=64, page=32, shared_lo=8192, shared_hi=8192, own_lo=20, own_hi=1501, pad=3),
        # five prompts answered several times each, in a cache of the model's own type
        prefix("prefix_groups_16bit", bits=16, batch=80, groups=5, heads=28, kv_heads=4, page=64, shared_lo=700, shared_hi=6007,
               own_lo=5, own_hi=701),
        # four drafted tokens of each sequence behind a long document: the most operations
        prefix("prefix_long_drafts", batch=48, heads=64, kv_heads=8, dim=64, page=128, new_lo=4, new_hi=4, shared_lo=32000,
               shared_hi=32000, own_lo=4, own_hi=2503),
        # one generated token of one sequence: latency counts
        linear("linear_one_token", key_heads=16),
        # a decoding batch, every state read and written
        linear("linear_step", type="f16", batch=96, pad=2),
        # drafted tokens in a state-space layer, one key head for all heads
        linear("linear_drafts", batch=24, heads=48, key_heads=1, dim=64, new_lo=2, new_hi=5),
        # ragged prompts, some behind tokens that were seen before, a decay for each head alone
        linear("linear_prompts", type="f16", batch=7, heads=16, key_heads=16, key_dim=64, dim=96, new_lo=301, new_hi=4099, each=False),
        # one long prompt from an empty state: the most bytes
        linear("linear_long_prompt", new_lo=16384, new_hi=16384, fresh=True),
        # the next token of one sequence: latency counts
        sample("sample_one"),
        # a decoding batch with filters of every kind, an odd vocabulary, rows of a wider buffer
        sample("sample_batch", type="bf16", rows=96, vocab=100003, min_p=True, greedy=True, pad=5),
        # many sequences, no top-k, some with most tokens forbidden
        sample("sample_many", type="f32", rows=320, vocab=200000, top_k=False, masked=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    kind = rng.choice(["prefix", "linear", "sample"])
    t = rng.choice(["f16", "bf16"])
    if kind == "prefix":
        while True:
            kv = rng.choice([1, 2, 4, 8])
            batch, hi, tail = _log(rng, 1, 96), _log(rng, 1, 32000), _log(rng, 1, 2503)
            new = rng.choice([1, 1, 1, 2, 4, 8])
            c = prefix(type=t, bits=rng.choice([8, 8, 16]), batch=batch, groups=min(batch, rng.choice([1, 1, 1, 2, 5, 9])),
                       heads=kv * rng.choice([1, 3, 4, 7, 8]), kv_heads=kv, dim=rng.choice([64, 80, 96, 128, 128, 256]),
                       page=rng.choice([16, 32, 64, 128]), new_lo=max(1, new // 2), new_hi=new, shared_lo=hi // rng.choice([1, 1, 4]),
                       shared_hi=hi, own_lo=max(new, tail // 8), own_hi=max(new, tail), pad=rng.choice([0, 0, 2, 9]))
            keys = c["groups"] * hi + batch * tail
            if keys * kv * c["dim"] * c["bits"] <= 130000 * 4 * 128 * 16 and batch * new * c["heads"] * (hi + tail) * c["dim"] <= 48 * 4 * 64 * 34000 * 64:
                return c
    if kind == "linear":
        while True:
            kh = rng.choice([1, 2, 4, 8, 16])
            new = _log(rng, 1, 16384) if rng.random() < 0.6 else rng.choice([1, 1, 2, 5])
            c = linear(type=t, batch=_log(rng, 1, 96), heads=kh * rng.choice([1, 1, 2, 3]), key_heads=kh,
                       key_dim=rng.choice([32, 64, 96, 128, 128, 256]), dim=rng.choice([32, 64, 80, 96, 128, 128, 256]),
                       new_lo=max(1, new // 4), new_hi=new, each=rng.random() < 0.7, fresh=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 7]))
            n = sum(_spread(c["batch"], c["new_lo"], c["new_hi"]))
            if n * c["heads"] * (c["key_dim"] + c["dim"]) <= 16384 * 32 * 256 and c["batch"] * new <= 40000 and \
                    c["batch"] * c["heads"] * c["key_dim"] * c["dim"] <= 96 * 32 * 128 * 128:
                return c
    while True:
        c = sample(type=rng.choice(["f16", "bf16", "f32"]), rows=_log(rng, 1, 512), vocab=_log(rng, 100, 262144),
                   top_k=rng.random() < 0.6, top_p=rng.random() < 0.7, min_p=rng.random() < 0.3, greedy=rng.random() < 0.3,
                   masked=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 8]))
        if c["rows"] * c["vocab"] <= 320 * 200000:
            return c


# ------------------------------------------------------------------------------ sizes
def _spread(n, lo, hi, shift=0.0):
    """n lengths between lo and hi, the first of them hi where shift is 0: fixed, and in no order."""
    return [lo + int(round((hi - lo) * (1.0 - (b * 0.6180339887498949 + shift) % 1.0))) for b in range(n)]


def _members(c):
    """First sequence of each group and the end: groups of nearly the same size."""
    return [g * c["batch"] // c["groups"] for g in range(c["groups"] + 1)]


def _cached(c):
    """(new tokens, shared tokens in whole pages, tokens in all) of each sequence."""
    first, each = _members(c), _spread(c["groups"], c["shared_lo"], c["shared_hi"])
    new, tail = _spread(c["batch"], c["new_lo"], c["new_hi"]), _spread(c["batch"], c["own_lo"], c["own_hi"], 0.21)
    shared = [n // c["page"] * c["page"] for g, n in enumerate(each) for _ in range(first[g + 1] - first[g])]
    return new, shared, [s + max(a, n) for a, n, s in zip(tail, new, shared)]


def work(case):
    c = case
    if c["kind"] == "prefix":
        new, shared, full = _cached(c)
        first = _members(c)
        keys = sum(f - s for f, s in zip(full, shared)) + sum(shared[first[g]] for g in range(c["groups"]))
        pairs = sum(n * f - n * (n - 1) // 2 for n, f in zip(new, full))
        scale = 8.0 / c["page"] if c["bits"] == 8 else 0
        return {"bytes": keys * c["kv_heads"] * (2 * c["dim"] * c["bits"] / 8 + scale) + 4 * keys / c["page"] +
                4 * sum(new) * c["heads"] * c["dim"], "flops": 4 * pairs * c["heads"] * c["dim"]}
    if c["kind"] == "linear":
        n = sum(_spread(c["batch"], c["new_lo"], c["new_hi"]))
        rows = 4 * n * (c["key_heads"] * c["key_dim"] + c["heads"] * c["dim"])
        state = 4 * c["batch"] * c["heads"] * c["key_dim"] * c["dim"]
        return {"bytes": rows + (4 * n * c["heads"] if c["each"] else 4 * c["heads"]) + state * (1 if c["fresh"] else 2),
                "flops": 4 * n * c["heads"] * c["key_dim"] * c["dim"]}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * (4 if c["type"] == "f32" else 2) + 24 * c["rows"], "flops": 4 * n}


# ------------------------------------------------------------------------------ inputs
def _scale8(amax):
    """The smallest power of two s with amax <= 448 s, at least 2^-32."""
    m, e = torch.frexp(amax / 448.0)
    return torch.ldexp(torch.ones_like(amax), e - (m == 0.5).to(e.dtype)).clamp(min=2.0 ** -32)


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
    got = []
    for pack in (_pack_keys, _pack_values):
        x = torch.randn((pages, c["kv_heads"], c["page"], c["dim"]), generator=gen, device=gen.device)
        x *= torch.exp2(0.5 * torch.randn((pages, c["kv_heads"], 1, 1), generator=gen, device=gen.device))
        if c["bits"] == 16:
            got += [pack(x.to(TYPES[c["type"]]), c), None]
        else:
            s = _scale8(x.abs().amax((2, 3)))
            got += [pack((x / s[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8), c).view(torch.float8_e4m3fn), s]
    return got


def _table(c, shared, full, gen):
    """(page of each sequence and place, pages in all): a group's first pages are the same, unused places -1."""
    page, first = c["page"], _members(c)
    head = [shared[first[g]] // page for g in range(c["groups"])]
    pages = sum(head) + sum(-(-f // page) - s // page for f, s in zip(full, shared)) + 2
    order = torch.randperm(pages, generator=gen, device=gen.device).to(torch.int32)
    width = max(-(-f // page) for f in full) + 1
    table = torch.full((c["batch"], width), -1, dtype=torch.int32, device=gen.device)
    at = 0
    for g in range(c["groups"]):
        table[first[g]:first[g + 1], :head[g]] = order[at:at + head[g]]
        at += head[g]
        for b in range(first[g], first[g + 1]):
            n = -(-full[b] // page) - head[g]
            table[b, head[g]:head[g] + n] = order[at:at + n]
            at += n
    return table, pages, width


def _ends(counts, dev):
    return torch.tensor(np.cumsum([0] + list(counts)), dtype=torch.int32, device=dev)


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    t = TYPES[c["type"]]
    randn = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, generator=gen, device=dev)  # noqa: E731
    s = {"case": c}
    if c["kind"] == "prefix":
        new, shared, full = _cached(c)
        rows = sum(new) + c["pad"]
        s["q"] = randn(rows, c["heads"], c["dim"]).to(t)
        s["cu"], s["lens"] = _ends(new, dev), torch.tensor(full, dtype=torch.int32, device=dev)
        s["group"] = torch.tensor(_members(c), dtype=torch.int32, device=dev)
        s["shared"] = torch.tensor([shared[b] for b in _members(c)[:-1]], dtype=torch.int32, device=dev)
        s["table"], s["pages"], s["width"] = _table(c, shared, full, gen)
        s["kc"], s["ks"], s["vc"], s["vs"] = _cache(c, s["pages"], gen)
        s["o"] = torch.zeros((rows, c["heads"], c["dim"]), dtype=t, device=dev)
        s["rows"], s["max_new"], s["max_len"], s["max_shared"] = rows, max(new), max(full), max(shared)
    elif c["kind"] == "linear":
        new = _spread(c["batch"], c["new_lo"], c["new_hi"])
        rows, h = sum(new) + c["pad"], c["heads"]
        s["q"] = randn(rows, c["key_heads"], c["key_dim"]).to(t)
        s["k"] = (randn(rows, c["key_heads"], c["key_dim"]) / math.sqrt(c["key_dim"])).to(t)
        s["v"] = randn(rows, h, c["dim"]).to(t)
        # heads that remember a few tokens and heads that remember thousands
        slow = torch.exp(torch.linspace(math.log(2e-4), math.log(2.0), h, device=dev))
        s["g"] = -slow * torch.nn.functional.softplus(randn(rows, h)) if c["each"] else -slow * (0.8 + 0.4 * rand(h))
        s["cu"] = _ends(new, dev)
        # a state is read from one slot and written to another; the slots stand in no order
        place = torch.randperm(2 * c["batch"], generator=gen, device=dev).to(torch.int32)
        s["from"], s["to"] = place[:c["batch"]].contiguous(), place[c["batch"]:].contiguous()
        if c["fresh"]:
            s["from"] = torch.full_like(s["from"], -1)
        s["state"] = randn(2 * c["batch"], h, c["key_dim"], c["dim"])
        s["o"] = torch.zeros((rows, h, c["dim"]), dtype=t, device=dev)
        s["rows"], s["max_new"] = rows, max(new)
    else:
        r, n = c["rows"], c["vocab"]
        x = randn(r, n + c["pad"]) * 2.2
        # a few likely tokens
        likely = torch.randint(0, n, (r, min(n, 64)), generator=gen, device=dev)
        x.scatter_add_(1, likely, 14.0 * rand(*likely.shape) ** 2)
        if c["masked"]:  # every fourth row may take some tokens only
            hide = rand(r, n + c["pad"]) < 0.98
            hide[torch.arange(r, device=dev) % 4 != 3] = False
            hide.scatter_(1, likely[:, :1], False)
            x.masked_fill_(hide, -math.inf)
        s["wide"] = x.to(t)
        s["x"] = s["wide"][:, :n]
        pick = lambda values: torch.tensor(values, device=dev)[torch.randint(0, len(values), (r,), generator=gen, device=dev)]  # noqa: E731
        s["temperature"] = 0.5 + 0.8 * rand(r)
        if c["greedy"]:
            s["temperature"] *= pick([0.0, 1.0, 1.0, 1.0])
        s["top_k"] = pick([0, 1, 20, 50, 1000]).to(torch.int32) if c["top_k"] else None
        s["top_p"] = pick([0.8, 0.9, 0.95, 1.0]) if c["top_p"] else None
        s["min_p"] = pick([0.0, 0.02, 0.1]) if c["min_p"] else None
        s["u"] = rand(r)
        s["token"] = torch.zeros(r, dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------------------ the plain forms
def _padded(x, cu, n):
    """[rows][heads][dim] -> [batch][heads][n][dim] in 32 bits, zeros behind a sequence's rows."""
    at = cu[:-1, None] + torch.arange(n, device=x.device)
    got = x[at.clamp(max=x.shape[0] - 1).long()].float() * (at < cu[1:, None])[:, :, None, None]
    return got.permute(0, 2, 1, 3)


def _places(cu, rows):
    """(sequence, index among its new rows) of each row; rows behind the last sequence get it too."""
    at = torch.arange(rows, device=cu.device, dtype=torch.int32)
    b = (torch.searchsorted(cu, at, right=True) - 1).clamp(0, cu.numel() - 2)
    return b, at - cu[b]


def _rows_of(o, s):
    """[batch][heads][n][dim] back to rows; those behind the last sequence stay."""
    seq, i = _places(s["cu"], s["rows"])
    got = o[seq, :, i.clamp(max=o.shape[2] - 1).long()].to(s["o"].dtype)
    return torch.where((torch.arange(s["rows"], device=o.device) < s["cu"][-1])[:, None, None], got, s["o"])


def _plain_prefix(s):
    """Every sequence reads all of its pages, a part of the batch at a time."""
    c = s["case"]
    n, kv, heads, d = s["max_new"], c["kv_heads"], c["heads"], c["dim"]
    q = _padded(s["q"], s["cu"], n)
    keys = s["width"] * c["page"]
    o = torch.empty_like(q)
    j = torch.arange(keys, device=q.device)
    per = max(1, (1 << 30) // (keys * (2 * kv * d + heads * n)))
    for b in range(0, c["batch"], per):
        part = slice(b, min(c["batch"], b + per))
        pages, lens = s["table"][part].clamp(min=0).long(), s["lens"][part]
        m = pages.shape[0]
        k, v = s["kc"], s["vc"]
        if c["bits"] == 8:
            k = k.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["ks"][pages][..., None, None, None, None]
            v = v.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["vs"][pages][..., None, None, None]
        else:
            k, v = k[pages].float(), v[pages].float()
        live = (j < lens[:, None])[:, None, :, None]
        k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(m, kv, keys, d) * live
        v = v.permute(0, 2, 1, 3, 5, 4).reshape(m, kv, keys, d) * live
        place = lens - (s["cu"][1:] - s["cu"][:-1])[part]
        seen = j <= (place[:, None] + torch.arange(n, device=q.device))[:, :, None]
        x = torch.matmul(q[part].reshape(m, kv, heads // kv * n, d), k.transpose(2, 3)).reshape(m, kv, heads // kv, n, keys)
        x = x.mul_(1.0 / math.sqrt(d)).masked_fill_(~seen[:, None, None], -math.inf)
        x = x.sub_(x.amax(-1, keepdim=True)).exp_()
        x = x.div_(x.sum(-1, keepdim=True)).reshape(m, kv, heads // kv * n, keys)
        o[part] = torch.matmul(x, v).reshape(m, heads, n, d)
    return _rows_of(o, s)


def _plain_linear(s):
    """Chunk after chunk for all sequences at once; rows that are not there have no key and keep the state."""
    c = s["case"]
    n, h, dev = s["max_new"], c["heads"], s["q"].device
    q, k, v = (_padded(s[x], s["cu"], n) for x in "qkv")
    rep = h // c["key_heads"]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    g = s["g"] if c["each"] else s["g"].expand(s["rows"], h)
    g = _padded(g[..., None], s["cu"], n)[..., 0].double()
    live = torch.arange(n, device=dev) < (s["cu"][1:] - s["cu"][:-1])[:, None]
    g = g * live[:, None]
    start = s["from"].long()
    state = s["state"][start.clamp(min=0)] * (start >= 0)[:, None, None, None]
    o = torch.empty_like(v)
    for at in range(0, n, CHUNK):
        part = slice(at, min(n, at + CHUNK))
        b = g[:, :, part].cumsum(-1)
        m = b.shape[-1]
        late = torch.ones(m, m, dtype=torch.bool, device=dev).tril()
        w = torch.where(late, torch.exp((b[..., :, None] - b[..., None, :]).float()), 0.0)
        x = torch.matmul(q[:, :, part], k[:, :, part].transpose(2, 3)) * w
        o[:, :, part] = torch.matmul(x, v[:, :, part]) + torch.exp(b).float()[..., None] * torch.matmul(q[:, :, part], state)
        left = torch.exp(b[..., -1:] - b).float()[..., None]
        state = torch.exp(b[..., -1]).float()[..., None, None] * state + torch.matmul(k[:, :, part].transpose(2, 3), left * v[:, :, part])
    s["state"][s["to"].long()] = state
    return _rows_of(o * (1.0 / math.sqrt(c["key_dim"])), s), s["state"]


def _plain_sample(s):
    """Sorted, cut and summed in 64 bits: tokens in descending order, ties by index."""
    x = s["x"].float()
    r, n = x.shape
    t = s["temperature"]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = order[:, 0]
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(t > 0, t, 1.0)[:, None].double())
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], n)
        w = torch.where(torch.arange(n, device=x.device) < k[:, None], w, 0.0)
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_p"] is not None:  # the fewest tokens whose sum reaches top_p of all: those before which it does not
        total = torch.cumsum(w, 1)
        keep[:, 1:] = total[:, :-1] < s["top_p"][:, None].double() * total[:, -1:]
        del total
    if s["min_p"] is not None:
        keep &= w >= s["min_p"][:, None].double()
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))  # in the order of the vocabulary
    total = torch.cumsum(w, 1)
    goal = s["u"][:, None].double() * total[:, -1:]
    token = (total <= goal).sum(1).clamp(max=n - 1)
    return torch.where(t > 0, token, greedy).to(torch.int32)


# ------------------------------------------------------------------------------ the framework's calls
def _plan(s, ops):
    """Descriptors and the workspace that a program makes once for its shapes."""
    c = s["case"]
    t = {"f16": ops.F16, "bf16": ops.BF16, "f32": 2}[c["type"]]
    strides = lambda x: (x.stride(0), x.stride(1))  # noqa: E731
    if c["kind"] == "prefix":
        cache = ops.cache_desc(t, c["bits"], c["kv_heads"], c["dim"], c["page"], s["pages"], s["width"])
        d = ops.prefix_attention_desc(cache, c["heads"], 1.0 / math.sqrt(c["dim"]), q=strides(s["q"]), o=strides(s["o"]),
                                      max_new=s["max_new"], max_len=s["max_len"], max_shared=s["max_shared"])
        need = ops.prefix_attention_workspace(d, c["batch"], c["groups"], s["rows"])
    elif c["kind"] == "linear":
        d = ops.linear_attention_desc(t, c["heads"], c["key_heads"], c["key_dim"], c["dim"], 1.0 / math.sqrt(c["key_dim"]),
                                      2 * c["batch"], q=strides(s["q"]), k=strides(s["k"]), v=strides(s["v"]), o=strides(s["o"]),
                                      g=strides(s["g"]) if c["each"] else (0, 1), max_new=s["max_new"])
        need = ops.linear_attention_workspace(d, c["batch"], s["rows"])
    else:
        d = ops.sample_desc(t, c["vocab"], row=s["x"].stride(0))
        need = ops.sample_workspace(d, c["rows"])
    return d, torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda"), need


def _own_run(s):
    from infvino_amd import ops
    c = s["case"]
    if "plan" not in s:
        s["plan"] = _plan(s, ops)
    d, space, need = s["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda *names: [None if s[x] is None else s[x].data_ptr() for x in names]  # noqa: E731
    if c["kind"] == "prefix":
        ops.prefix_attention(d, *at("q", "kc", "vc", "ks", "vs", "cu", "lens", "table", "group", "shared", "o"), c["batch"],
                             c["groups"], s["rows"], space.data_ptr(), need, stream)
        return s["o"]
    if c["kind"] == "linear":
        ops.linear_attention(d, *at("q", "k", "v", "g", "cu", "from", "to", "state", "o"), c["batch"], s["rows"], space.data_ptr(),
                             need, stream)
        return s["o"], s["state"]
    ops.sample(d, *at("x", "temperature", "top_k", "top_p", "min_p", "u", "token"), c["rows"], space.data_ptr(), need, stream)
    return s["token"]


def run(state):
    if own:
        return _own_run(state)
    return {"prefix": _plain_prefix, "linear": _plain_linear, "sample": _plain_sample}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------ in 64 bits
def _exact_prefix(s):
    """Sequence by sequence, page by page."""
    c = s["case"]
    h, n, d, group = c["kv_heads"], c["page"], c["dim"], c["heads"] // c["kv_heads"]
    kc = s["kc"].permute(0, 1, 2, 4, 3, 5).reshape(-1, h, n, d)
    vc = s["vc"].permute(0, 1, 2, 4, 3).reshape(-1, h, n, d)
    o, row = s["o"].double(), 0
    for b, (new, full) in enumerate(zip(*_cached(c)[::2])):
        pages = s["table"][b, :-(-full // n)].long()
        k, v = (x.view(torch.uint8)[pages].view(x.dtype) if c["bits"] == 8 else x[pages] for x in (kc, vc))
        k, v = k.double(), v.double()
        if c["bits"] == 8:
            k, v = k * s["ks"][pages].double()[:, :, None, None], v * s["vs"][pages].double()[:, :, None, None]
        k, v = (x.transpose(0, 1).reshape(h, -1, d)[:, :full] for x in (k, v))
        late = torch.arange(full, device=o.device) > torch.arange(full - new, full, device=o.device)[:, None]
        for kh in range(h):
            q = s["q"][row:row + new, kh * group:(kh + 1) * group].double().transpose(0, 1)
            x = (q @ k[kh].t() / math.sqrt(d)).masked_fill(late, -math.inf)
            o[row:row + new, kh * group:(kh + 1) * group] = (torch.softmax(x, -1) @ v[kh]).transpose(0, 1)
        row += new
    return o


def _exact_linear(s):
    """Every pair of tokens, head by head: o_t = sum over s <= t of e^(b_t - b_s) (q_t k_s) v_s, and the first state's part."""
    c = s["case"]
    o, state, row = s["o"].double(), s["state"].double(), 0
    rep, scale = c["heads"] // c["key_heads"], 1.0 / math.sqrt(c["key_dim"])
    start, to = s["from"].tolist(), s["to"].tolist()
    got = state.clone()
    for i, n in enumerate(_spread(c["batch"], c["new_lo"], c["new_hi"])):
        rows = slice(row, row + n)
        g = s["g"][rows].double() if c["each"] else s["g"].double().expand(n, -1)
        b = g.cumsum(0)
        for h in range(c["heads"]):
            q, k, v = s["q"][rows, h // rep].double(), s["k"][rows, h // rep].double(), s["v"][rows, h].double()
            first = state[start[i], h] if start[i] >= 0 else torch.zeros_like(state[0, h])
            for at in range(0, n, 2048):
                end = min(n, at + 2048)
                age = b[at:end, h, None] - b[None, :end, h]
                seen = torch.arange(end, device=o.device) <= torch.arange(at, end, device=o.device)[:, None]
                x = (q[at:end] @ k[:end].t()) * torch.exp(age.masked_fill(~seen, -math.inf))
                o[row + at:row + end, h] = scale * (x @ v[:end] + torch.exp(b[at:end, h, None]) * (q[at:end] @ first))
            got[to[i], h] = torch.exp(b[-1, h]) * first + (k * torch.exp(b[-1, h] - b[:, h])[:, None]).t() @ v
        row += n
    return o, got


def _exact_sample(s):
    """Row by row: tokens ordered by one whole number of score and index."""
    n = s["case"]["vocab"]
    index = torch.arange(n, device=s["x"].device)
    rows = []
    value = lambda name, i: None if s[name] is None else float(s[name][i])  # noqa: E731
    for i in range(s["case"]["rows"]):
        x = s["x"][i].float() + 0.0
        bits = x.view(torch.int32).long()
        order = (torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 20 - index).argsort(descending=True)
        t = value("temperature", i)
        if t <= 0:
            rows.append(int(order[0]))
            continue
        y = x.double()[order]
        w = torch.exp((y - y[0]) / t)
        count, k = n, value("top_k", i)
        if k is not None and 0 < k < n:
            count = int(k)
        if s["top_p"] is not None:
            sums = w[:count].cumsum(0)
            reached = (sums >= value("top_p", i) * sums[-1]).nonzero()
            count = int(reached[0]) + 1 if len(reached) else count
        if s["min_p"] is not None:
            count = max(1, min(count, int((w >= value("min_p", i)).sum())))
        kept, _ = order[:count].sort()
        sums = torch.exp((x.double()[kept] - y[0]) / t).cumsum(0)
        beyond = (sums > value("u", i) * sums[-1]).nonzero()
        rows.append(int(kept[beyond[0, 0]]))
    return torch.tensor(rows, dtype=torch.int32, device=s["x"].device)


def exact(case, seed):
    s = prepare(case, seed)
    return {"prefix": _exact_prefix, "linear": _exact_linear, "sample": _exact_sample}[s["case"]["kind"]](s)
