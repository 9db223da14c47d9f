"""Sequence operators on the GPU against their definitions in 64 bits: rotary positions, appending to a
paged cache, attention over it and over ragged rows.

Tolerances (u = half a step of the type relative to the value: 2^-11 fp16, 2^-8 bf16):
  rotation   u |y| for the rounding, 2^-21 (|a| + |b|) for the products, the sum, and the sine and
             cosine in fp32 (8 roundings of 2^-24), 2^-25 for fp16's subnormal values
  8-bit      half a step of e4m3, 2^-4 |y|, or of its subnormal values, 2^-10 of the scale, and
             the rotation's fp32 error
  attention  u |o| for the output; the weights are rounded to the type: u sum w |v|; fp32 scores
             are off by dim 2^-24 sum |q k| scale and exponents by 2^-15 at most (|t| <= 2^8 in
             units of log 2, rounded to 2^-24 of that), which moves the output by twice that times sum w |v|; fp16 weights
             below 2^-24 of the largest are off by 2^-25 each: keys 2^-25 max |v|
"""
import math

import pytest
import torch

from infvino_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f16": (ops.F16, torch.float16, 2.0 ** -11), "bf16": (ops.BF16, torch.bfloat16, 2.0 ** -8)}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, t, *shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(t)


def _p(x):
    return None if x is None else x.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _ends(counts):
    e = [0]
    for n in counts:
        e.append(e[-1] + n)
    return _i32(e)


# ------------------------------------------------------------------ rotation
def _axis_of(sections, dealt):
    half, axes = sum(sections), len(sections)
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [f % axes if f % axes and f // axes < sections[f % axes] else 0 for f in range(half)]


def _rotated(x, pos, freq, sections, adjacent, dealt):
    """(x [tokens][heads][dim] rotated, |a| + |b| of each channel's pair), in 64 bits."""
    x = x.double()
    half = sum(sections)
    ang = pos.double()[torch.tensor(_axis_of(sections, dealt), device="cuda")].t() * freq.double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    if adjacent:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    y, m = x.clone(), x.abs()
    u, w, n = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    if adjacent:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = u, w
        m[..., 0:2 * half:2], m[..., 1:2 * half:2] = n, n
    else:
        y[..., :half], y[..., half:2 * half] = u, w
        m[..., :half], m[..., half:2 * half] = n, n
    return y, m


def _freq(half):
    return torch.tensor([10000.0 ** (-f / half) for f in range(half)], dtype=torch.float32, device="cuda")


ROPES = [  # tokens, heads, dim, sections, adjacent, dealt
    (1, 1, 8, (4,), False, False), (1, 40, 128, (64,), False, False), (1, 3, 8, (4,), True, False),
    (3, 5, 72, (36,), False, False), (17, 7, 80, (20, 20), False, False), (33, 2, 80, (40,), True, False),
    (129, 16, 128, (24, 20, 20), False, True), (65, 4, 128, (16, 24, 24), True, True), (40, 3, 96, (8, 4, 4, 8), False, False),
    (31, 9, 256, (32,), False, False), (12, 3, 256, (12, 12, 8), True, True), (1000, 8, 64, (32,), True, False),
    (7, 2, 1024, (512,), False, False), (5, 4096, 16, (8,), False, False), (2500, 40, 128, (64,), False, False),
    (6, 2, 128, (60, 4), False, True), (4, 3, 104, (44,), False, False),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,heads,dim,sections,adjacent,dealt", ROPES)
def test_rope(t, tokens, heads, dim, sections, adjacent, dealt):
    code, dt, u = TYPES[t]
    g = _gen(tokens + dim)
    x = _randn(g, dt, tokens, heads, dim)
    pos = torch.randint(-50, 1000000, (len(sections), tokens), generator=g, device="cuda", dtype=torch.int32)
    freq = _freq(sum(sections))
    y = torch.full_like(x, 7.0)
    d = ops.rope_desc(code, heads, dim, sections, adjacent=adjacent, dealt=dealt, pos_axis=tokens)
    ops.rope(d, _p(x), _p(pos), _p(freq), _p(y), tokens, _stream())
    ref, mag = _rotated(x, pos, freq, sections, adjacent, dealt)
    rot = 2 * sum(sections)
    assert ((y.double() - ref).abs() <= u * ref.abs() + 2.0 ** -21 * mag + 2.0 ** -25)[..., :rot].all()
    assert torch.equal(y[..., rot:], x[..., rot:])
    # in place: the same bits
    z = x.clone()
    ops.rope(d, _p(z), _p(pos), _p(freq), _p(z), tokens, _stream())
    assert torch.equal(z.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("lo,hi", [((1 << 22) - 40, (1 << 22) + 40), (-(1 << 22) - 40, 40 - (1 << 22)), (1 << 24, (1 << 24) + 80),
                                   ((1 << 31) - 80, (1 << 31) - 1), (-(1 << 31), 80 - (1 << 31))])
def test_rope_far_positions(lo, hi):
    """Angles of positions up to 32 bits: fp32 inputs of 1 and 0 through bf16's own rounding would hide an error, so values
    that f16 has exactly; 64 bits carry 2 pi x 2^31 turns to 2^-19, which bounds the last two."""
    code, dt, u = TYPES["f16"]
    pos = torch.arange(lo, hi, dtype=torch.int64, device="cuda").to(torch.int32).reshape(1, -1)
    n = pos.shape[1]
    x = torch.ones((n, 1, 128), dtype=dt, device="cuda")
    y, freq = torch.empty_like(x), _freq(64)
    ops.rope(ops.rope_desc(code, 1, 128, (64,)), _p(x), _p(pos), _p(freq), _p(y), n, _stream())
    ref, mag = _rotated(x, pos, freq, (64,), False, False)
    assert ((y.double() - ref).abs() <= u * ref.abs() + 2.0 ** -18 * mag + 2.0 ** -25).all()


def test_rope_strided_rows():
    """q and k of packed q, k, v rows, written head by head; 8-byte row starts."""
    code, dt, u = TYPES["bf16"]
    for tokens, heads, dim, pad in ((37, 6, 64, 0), (21, 4, 128, 4), (9, 5, 72, 12)):
        g = _gen(dim)
        rows = _randn(g, dt, tokens, heads * dim * 2 + pad)
        out = torch.full((heads, tokens, dim), 3.0, dtype=dt, device="cuda")
        pos = torch.arange(tokens, dtype=torch.int32, device="cuda").reshape(1, tokens) * 3
        freq = _freq(dim // 2)
        d = ops.rope_desc(code, heads, dim, (dim // 2,), x=(rows.stride(0), dim), y=(dim, tokens * dim))
        ops.rope(d, _p(rows), _p(pos), _p(freq), _p(out), tokens, _stream())
        ref, mag = _rotated(rows[:, :heads * dim].unflatten(1, (heads, dim)), pos, freq, (dim // 2,), False, False)
        got = out.permute(1, 0, 2).double()
        assert ((got - ref).abs() <= u * ref.abs() + 2.0 ** -21 * mag).all()


def test_rope_leaves_other_memory_alone():
    code, dt, _ = TYPES["f16"]
    buf = torch.full((5, 4, 48), 9.0, dtype=dt, device="cuda")
    x = torch.ones((5, 4, 32), dtype=dt, device="cuda")
    pos, freq = torch.zeros((1, 5), dtype=torch.int32, device="cuda"), _freq(16)
    d = ops.rope_desc(code, 4, 32, (16,), y=(4 * 48, 48))
    ops.rope(d, _p(x), _p(pos), _p(freq), _p(buf), 3, _stream())
    assert (buf[:3, :, :32] == 1).all() and (buf[:3, :, 32:] == 9).all() and (buf[3:] == 9).all()


# ------------------------------------------------------------------ the cache
class Cache:
    """A paged cache and its plain view."""

    def __init__(self, t, bits, heads, dim, page, pages, width):
        self.code, self.dt, self.u = TYPES[t]
        self.bits, self.heads, self.dim, self.page, self.pages, self.width = bits, heads, dim, page, pages, width
        self.desc = ops.cache_desc(self.code, bits, heads, dim, page, pages, width)
        nb, ns = ops.cache_bytes(self.desc)
        # NaN everywhere: a page's empty slots may hold anything
        self.kc = torch.full((nb,), 0x7f if bits == 8 else 0xff, dtype=torch.uint8, device="cuda")
        self.vc = self.kc.clone()
        self.ks = torch.full((ns // 4,), math.nan, device="cuda") if bits == 8 else None
        self.vs = self.ks.clone() if bits == 8 else None

    def values(self):
        """keys, values as [pages][heads][page][dim] codes in 64 bits, without scales."""
        e = 16 if self.bits == 8 else 8
        dt = torch.float8_e4m3fn if self.bits == 8 else self.dt
        k = self.kc.view(dt).reshape(self.pages, self.heads, self.page // 4, self.dim // e, 4, e)
        v = self.vc.view(dt).reshape(self.pages, self.heads, self.page // e, self.dim, e)
        return (k.double().permute(0, 1, 2, 4, 3, 5).reshape(self.pages, self.heads, self.page, self.dim),
                v.double().permute(0, 1, 2, 4, 3).reshape(self.pages, self.heads, self.page, self.dim))

    def scales(self):
        return [s.double().reshape(self.pages, self.heads) for s in (self.ks, self.vs)]

    def rows(self, table, n):
        """keys, values [n][heads][dim] of one sequence, in 64 bits."""
        k, v = self.values()
        if self.bits == 8:
            ks, vs = self.scales()
            k, v = k * ks[..., None, None], v * vs[..., None, None]
        ids = torch.tensor(table[:-(-n // self.page)] or [0], device="cuda")
        return [x[ids].permute(1, 0, 2, 3).reshape(self.heads, -1, self.dim)[:, :n].permute(1, 0, 2) for x in (k, v)]

    def append(self, k, v, pos, freq, cu, lens, table, batch, sections=(), adjacent=False, dealt=False, k_strides=None, v_strides=None):
        d = ops.append_desc(self.desc, sections, adjacent=adjacent, dealt=dealt, k=k_strides, v=v_strides,
                            pos_axis=0 if pos is None else pos.stride(0))
        ops.kv_append(d, _p(k), _p(v), _p(pos), _p(freq), _p(cu), _p(lens), _p(table), _p(self.kc), _p(self.vc), _p(self.ks),
                      _p(self.vs), batch, k.shape[0], _stream())


def _e4m3(x):
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _pow2_scale(amax):
    return torch.exp2(torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** -32))))


def _tables(gen, used, width, pages):
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    out, at = [], 0
    for n in used:
        out.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return out


APPENDS = [  # bits, heads, dim, page, sections, adjacent, dealt, chunks of each sequence
    (8, 2, 64, 16, (32,), False, False, [(1, 1, 1, 1), (15, 1, 1, 16), (0, 3, 0, 40)]),
    (8, 1, 128, 16, (24, 20, 20), False, True, [(5, 11, 17), (33, 1, 2)]),
    (8, 3, 80, 32, (20, 20), True, False, [(70, 1, 5), (0, 0, 1), (31, 33, 64)]),
    (8, 2, 256, 128, (16,), False, False, [(130, 1, 300), (1, 127, 1)]),
    (8, 2, 96, 64, (), False, False, [(64, 1, 63), (100, 28, 1)]),
    (8, 4, 16, 16, (4,), False, False, [(3, 30, 1)]),
    (16, 2, 64, 16, (32,), False, False, [(1, 1, 1, 1), (15, 1, 1, 16), (0, 3, 0, 40)]),
    (16, 3, 80, 32, (20, 20), True, False, [(70, 1, 5), (0, 0, 1), (31, 33, 64)]),
    (16, 2, 256, 128, (64, 64), False, True, [(130, 1, 300), (1, 127, 1)]),
    (16, 1, 112, 64, (), False, False, [(65, 64, 1)]),
    # runs of 4 and 8 channels, whole pages of many channels
    (8, 2, 240, 128, (12,), False, False, [(128, 1, 200), (3, 0, 125)]),
    (8, 2, 240, 64, (8, 8, 8), True, True, [(70, 30)]),
    (8, 1, 256, 128, (24, 16), False, True, [(300, 1)]),
    (8, 1, 192, 128, (64,), True, False, [(129, 129)]),
    (16, 2, 144, 16, (4, 8), False, False, [(20, 13)]),
    # many sequences, some of them without new tokens
    (8, 2, 64, 16, (32,), False, False, [(i % 5, i % 3 == 0, 1) for i in range(63)]),
    (8, 1, 128, 32, (24, 20, 20), False, True, [(i % 41, i % 3, 1) for i in range(70)]),
    (8, 3, 32, 64, (), False, False, [(0 if i % 7 else 70, 1, 2) for i in range(130)]),
    (16, 2, 64, 16, (32,), True, False, [(i % 19, i % 2, 1) for i in range(200)]),
    (8, 4, 128, 64, (32,), False, False, [(i % 7 and 3 + i % 90, i % 3, 3, 60 * (i == 5)) for i in range(70)]),
    (8, 4, 96, 64, (16, 32), False, True, [(i % 7 and 3 + i % 64, i % 3, 3) for i in range(66)]),
    (8, 8, 64, 128, (), False, False, [(i % 5 and 3 + i % 150, i % 3, 3) for i in range(40)]),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits,heads,dim,page,sections,adjacent,dealt,chunks", APPENDS)
def test_append(t, bits, heads, dim, page, sections, adjacent, dealt, chunks):
    """Chunk after chunk of every sequence; after each the whole cache against the definition, older
    tokens' codes and everything that is no sequence's included."""
    code, dt, u = TYPES[t]
    g = _gen(dim + page)
    batch, rounds = len(chunks), len(chunks[0])
    used = [-(-sum(c) // page) for c in chunks]
    width, pages = max(used) + 1, sum(used) + 2
    table = _tables(g, used, width, pages)
    cache = Cache(t, bits, heads, dim, page, pages, width)
    ref = list(cache.values())  # what the cache should hold
    refs = cache.scales() if bits == 8 else None
    old = [0] * batch
    freq = _freq(max(1, sum(sections)))
    for n in range(rounds):
        new = [c[n] for c in chunks]
        rows = sum(new) + 2  # two rows of padding
        # magnitudes that grow, so that scales of half-filled pages have to as well
        k, v = (_randn(g, dt, rows, heads, dim, scale=s) for s in (2.0 ** n, 1.5 ** n))
        pos = torch.randint(0, 100000, (max(1, len(sections)), rows), generator=g, device="cuda", dtype=torch.int32)
        full = [a + b for a, b in zip(old, new)]
        cache.append(k, v, pos, freq, _ends(new), _i32(full), _i32(table), batch, sections, adjacent, dealt)
        kr, mag = _rotated(k, pos, freq, sections, adjacent, dealt) if sections else (k.double(), 0 * k.double())
        fresh = torch.zeros((pages, heads, page, dim), dtype=torch.bool, device="cuda")
        slack = [torch.zeros((pages, heads, page, dim), dtype=torch.double, device="cuda") for _ in range(2)]
        row = 0
        for b in range(batch):
            at = old[b]
            while at < full[b]:
                id, lo = table[b][at // page], at % page
                hi = min(page, lo + full[b] - at)
                for i, (x, m) in enumerate(((kr, mag), (v.double(), None))):
                    part = x[row:row + hi - lo].transpose(0, 1)
                    err = 0 if m is None else 2.0 ** -21 * m[row:row + hi - lo].transpose(0, 1)
                    if bits == 16:
                        ref[i][id, :, lo:hi] = part
                        slack[i][id, :, lo:hi] = (u * part.abs() + err + 2.0 ** -25) if m is not None else 0
                        continue
                    s = _pow2_scale(part.abs().amax((1, 2)))
                    if lo:
                        s = torch.maximum(s, refs[i][id])
                        ref[i][id] = _e4m3(ref[i][id] * (refs[i][id] / s)[:, None, None])
                    refs[i][id] = s
                    y = part / s[:, None, None]
                    ref[i][id, :, lo:hi] = y
                    slack[i][id, :, lo:hi] = 2.0 ** -4 * y.abs() + 2.0 ** -10 + err / s[:, None, None]
                fresh[id, :, lo:hi] = True
                row, at = row + hi - lo, at + hi - lo
        got = cache.values()
        for i in range(2):
            same = (got[i] == ref[i]) | (got[i].isnan() & ref[i].isnan())
            assert (same | fresh).all(), "older codes or slots of no token changed"
            assert ((got[i] - ref[i]).abs() <= slack[i])[fresh].all()
            if bits == 8:  # and nearly all codes are the nearest, not just near
                assert (got[i] == _e4m3(ref[i]))[fresh].double().mean() > 0.999 if fresh.any() else True
            ref[i] = torch.where(fresh, got[i], ref[i])
        if bits == 8:
            for a, b in zip(cache.scales(), refs):
                assert torch.equal(a.nan_to_num(-1), b.nan_to_num(-1))
        old = full


def test_append_twice_is_append_once():
    """The same call again (a replayed graph) leaves the same cache."""
    g = _gen(3)
    cache = Cache("bf16", 8, 2, 64, 32, 8, 5)
    table = _i32(_tables(g, [4, 3], 5, 8))
    k, v = _randn(g, torch.bfloat16, 100, 2, 64), _randn(g, torch.bfloat16, 100, 2, 64)
    cache.append(k, v, None, None, _ends([60, 40]), _i32([60, 40]), table, 2)
    args = (k * 3, v * 5, None, None, _ends([33, 7]), _i32([93, 47]), table, 2)
    cache.append(*args)
    once = [x.clone() for x in (cache.kc, cache.vc, cache.ks, cache.vs)]
    for _ in range(3):
        cache.append(*args)
        for a, b in zip(once, (cache.kc, cache.vc, cache.ks, cache.vs)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_odd_values_and_places():
    """Infinities and NaN, zeros, tiny and huge values; page numbers outside the cache; tokens behind the
    table's end and lengths shorter than the new tokens are dropped."""
    t = torch.bfloat16
    cache = Cache("bf16", 8, 1, 16, 16, 4, 2)
    x = torch.zeros((16, 1, 16), dtype=t, device="cuda")
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 2], x[3, 0, 3] = math.inf, -math.inf, math.nan, 100.0
    cache.append(x, x, None, None, _ends([16]), _i32([16]), _i32([[2, -1]]), 1)
    k, v = cache.values()
    for y, s in ((k[2, 0], cache.scales()[0][2, 0]), (v[2, 0], cache.scales()[1][2, 0])):
        # 100 / 0.25 lies between 384 and 416: to the even one
        assert s == 0.25 and y[0, 0] == 448 and y[1, 1] == -448 and y[2, 2].isnan() and y[3, 3] == 384
        y[2, 2] = 0
        assert y.isfinite().all() and (y != 0).sum() == 3
    for val, scale in ((0.0, 2.0 ** -32), (2.0 ** -40, 2.0 ** -32), (3.0e38, 2.0 ** 120), (448.0, 1.0), (450.0, 2.0)):
        y = torch.full((16, 1, 16), val, dtype=t, device="cuda")
        cache.append(y, y, None, None, _ends([16]), _i32([16]), _i32([[1, -1]]), 1)
        assert cache.scales()[0][1, 0] == scale and cache.scales()[1][1, 0] == scale
        want = _e4m3(y[0, 0, 0].double() / scale)
        assert (cache.values()[0][1] == want).all() and (cache.values()[1][1] == want).all()
    before = [z.clone() for z in (cache.kc, cache.vc)]
    y = torch.ones((16, 1, 16), dtype=t, device="cuda")
    for table, lens in (([[-1, 7]], 20), ([[4, 1 << 30]], 20), ([[3, 3]], 60), ([[0, 0]], -3), ([[0, 0]], 0)):  # tokens 44..59 lie behind two pages
        cache.append(y, y, None, None, _ends([16]), _i32([lens]), _i32(table), 1)
        assert torch.equal(cache.kc, before[0]) and torch.equal(cache.vc, before[1])
    # a length of 5 with 16 new rows: the last 5 are tokens 0..4
    z = torch.arange(16, device="cuda").reshape(16, 1, 1).expand(16, 1, 16).to(t).contiguous()
    cache.append(z, z, None, None, _ends([16]), _i32([5]), _i32([[0, -1]]), 1)
    k, s = cache.values()[0][0, 0], cache.scales()[0][0, 0]
    assert (k[:5, 0] * s).tolist() == [11, 12, 13, 14, 15] and k[5:].isnan().all()


def test_append_strided_rows():
    """Keys and values cut from packed q, k, v rows."""
    g = _gen(8)
    cache, plain = (Cache("f16", 8, 2, 64, 16, 6, 6) for _ in range(2))
    table = _i32(_tables(g, [5], 6, 6))
    rows = _randn(g, torch.float16, 70, 6 * 64 + 4)
    k, v = (rows[:, a:a + 128].unflatten(1, (2, 64)) for a in (128, 256))
    pos, freq = torch.arange(70, dtype=torch.int32, device="cuda").reshape(1, 70), _freq(32)
    cache.append(k, v, pos, freq, _ends([70]), _i32([70]), table, 1, (32,), k_strides=(rows.stride(0), 64), v_strides=(rows.stride(0), 64))
    plain.append(k.contiguous(), v.contiguous(), pos, freq, _ends([70]), _i32([70]), table, 1, (32,))
    assert torch.equal(cache.kc, plain.kc) and torch.equal(cache.vc, plain.vc)


# ------------------------------------------------------------------ attention
def _attend(q, k, v, place, causal, window, sinks, scale):
    """One sequence in 64 bits: q [n][heads][d], k and v [m][kv][d]; (o, sum w |v|, score error, weights' sum)."""
    q, k, v = q.double(), k.double(), v.double()
    n, heads, d = q.shape
    m, kv = k.shape[0], k.shape[1]
    if n == 0 or m == 0:
        z = torch.zeros_like(q)
        return z, z, torch.zeros((n, heads, 1), dtype=torch.double, device="cuda")
    k, v = (x.repeat_interleave(heads // kv, 1).transpose(0, 1) for x in (k, v))
    qh = q.transpose(0, 1)
    i, j = place[:, None], torch.arange(m, device="cuda")[None]
    see = torch.ones((n, m), dtype=torch.bool, device="cuda")
    if causal:
        see &= j <= i
    if window:
        see &= ((i - j).abs() < window) | (j < sinks)
    x = (qh @ k.transpose(1, 2)) * scale
    x = torch.where(see, x, -math.inf)
    w = (x - x.amax(-1, keepdim=True).clamp(min=-1e300)).exp()
    w = torch.where(see, w, 0.0)
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    err = d * 2.0 ** -24 * abs(scale) * torch.where(see, qh.abs() @ k.abs().transpose(1, 2), 0.0).amax(-1, keepdim=True)
    clean = torch.where(v.isfinite(), v, 0.0)
    o = w @ clean
    for c in (v == math.inf, v == -math.inf, v.isnan()):
        if c.any():  # an infinity or NaN reaches exactly the rows that see it
            hit = (see.double() @ c.double()) > 0
            val = torch.where(c, v, 0.0).nan_to_num(nan=0.0, posinf=1, neginf=-1).sum()
            o = torch.where(hit, math.nan if val == 0 else math.copysign(math.inf, float(val)) + o, o)
    return o.transpose(0, 1), (w @ clean.abs()).transpose(0, 1), err.transpose(0, 1)


def _close(got, o, av, err, u, keys, vmax):
    fine = o.isfinite()
    assert torch.equal(got.double().isfinite(), fine), "infinities and NaN reach other rows than see them"
    tol = u * o.abs() + u * av + 2 * (err + 2.0 ** -15) * av + keys * 2.0 ** -25 * vmax + 2.0 ** -25
    bad = ((got.double() - o).abs() > tol) & fine
    if bad.any():
        at = bad.nonzero()[0].tolist()
        print("first off at", at, "of", list(o.shape), got[tuple(at)].item(), o[tuple(at)].item(), "count", int(bad.sum()))
    assert not bad.any()


def _fill(cache, gen, table, lens, scale=1.0):
    """Caches `lens` tokens of each sequence by the append."""
    rows = sum(lens)
    if not rows:
        return
    k, v = (_randn(gen, cache.dt, rows, cache.heads, cache.dim, scale=scale) for _ in range(2))
    # every token of its own magnitude: pages have different scales
    v *= torch.exp2(torch.randint(-3, 4, (rows, 1, 1), generator=gen, device="cuda").float()).to(cache.dt)
    cache.append(k, v, None, None, _ends(lens), _i32(lens), _i32(table), len(lens))


def _run_paged(cache, q, cu, lens, table, heads, batch, window=0, sinks=0, max_new=0, max_len=0, o=None, scale=None):
    scale = 1 / math.sqrt(cache.dim) if scale is None else scale
    o = torch.full_like(q, 5.0) if o is None else o
    d = ops.paged_attention_desc(cache.desc, heads, scale, window, sinks, max_new=max_new, max_len=max_len)
    n = ops.paged_attention_workspace(d, batch, q.shape[0])
    ws = torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")  # NaN: its contents do not matter
    ops.paged_attention(d, _p(q), _p(cache.kc), _p(cache.vc), _p(cache.ks), _p(cache.vs), _p(cu), _p(lens), _p(table), _p(o), batch,
                        q.shape[0], _p(ws), n, _stream())
    return o, n


def _check_paged(cache, q, o, new, lens, table, window, sinks, scale=None):
    scale = 1 / math.sqrt(cache.dim) if scale is None else scale
    row = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        k, v = cache.rows(table[b], m)
        place = torch.arange(m - n, m, device="cuda")
        r, av, err = _attend(q[row:row + n], k, v, place, True, window, sinks, scale)
        vmax = torch.where(v.isfinite(), v, 0.0).abs().max() if m else 0
        _close(o[row:row + n], r, av, err, cache.u, m, vmax)
        row += n
    assert (o[row:] == 5.0).all(), "rows of no sequence changed"


PAGED = [  # bits, heads, kv heads, dim, page, new, lens, window, sinks
    (8, 8, 2, 128, 16, [1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 130], 0, 0),
    (8, 8, 8, 64, 32, [1, 1, 0, 1], [700, 1, 40, 257], 0, 0),
    (8, 28, 4, 128, 64, [1, 1], [1000, 129], 0, 0),
    (8, 32, 2, 80, 16, [1, 2, 3], [300, 2, 77], 0, 0),
    (8, 6, 2, 96, 128, [5, 5], [500, 5], 0, 0),
    (8, 16, 2, 256, 32, [1, 4], [400, 33], 0, 0),
    (8, 8, 2, 128, 16, [40, 1, 90], [200, 90, 90], 0, 0),
    (8, 8, 1, 64, 16, [300], [1000], 0, 0),
    (8, 4, 4, 16, 16, [1, 7], [100, 20], 0, 0),
    (8, 8, 2, 128, 32, [1, 1, 1, 5], [900, 100, 10, 400], 64, 4),
    (8, 8, 2, 128, 16, [50, 3], [600, 70], 33, 100),
    (8, 8, 2, 64, 64, [1, 2], [500, 300], 1, 0),
    (8, 4, 1, 128, 16, [1, 9], [500, 300], 17, 1),
    (8, 8, 2, 128, 16, [70], [400], 100, 3),
    (16, 8, 2, 128, 16, [1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 130], 0, 0),
    (16, 12, 4, 80, 32, [1, 4, 0, 17], [700, 50, 40, 257], 0, 0),
    (16, 16, 2, 256, 64, [1, 4], [400, 33], 0, 0),
    (16, 8, 1, 64, 16, [300], [700], 0, 0),
    (16, 8, 4, 256, 32, [40, 3], [500, 70], 33, 10),
    (16, 4, 1, 112, 16, [1, 9], [500, 300], 17, 1),
    # batches that fill the chip, whose waves take rows: four row ranges, then two
    (8, 8, 8, 128, 16, [70, 65] + [1, 0, 17] * 4, [300, 65] + [1, 40, 190] * 4, 0, 0),
    (8, 8, 8, 128, 64, [70] + [2] * 13, [500] + [290] * 13, 50, 3),
    (8, 8, 8, 80, 32, [80, 3] * 7, [80, 400] * 7, 0, 0),
    (8, 8, 8, 64, 32, [100] + [5] * 23, [400] + [131] * 23, 0, 0),
    (8, 8, 8, 256, 16, [70] + [1] * 13, [270] + [33] * 13, 0, 0),
    (16, 8, 8, 128, 16, [70, 65] + [1, 0, 17] * 4, [300, 65] + [1, 40, 190] * 4, 0, 0),
    (16, 8, 8, 64, 32, [100] + [5] * 23, [400] + [131] * 23, 70, 0),
    (16, 8, 8, 256, 16, [70] + [1] * 13, [270] + [33] * 13, 0, 0),
    (8, 32, 8, 128, 16, [5, 1, 0, 8] * 9, [40, 17, 3, 200] * 9, 0, 0),
    (8, 32, 8, 64, 16, [9, 1, 0, 16] * 9, [40, 17, 3, 200] * 9, 20, 2),
    (8, 32, 8, 240, 16, [5, 1, 0, 8] * 9, [40, 17, 3, 200] * 9, 0, 0),
    (16, 32, 8, 128, 16, [5, 1, 0, 8] * 9, [40, 17, 3, 200] * 9, 0, 0),
    (16, 32, 8, 64, 16, [9, 1, 0, 16] * 9, [40, 17, 3, 200] * 9, 0, 0),
    (16, 32, 8, 256, 16, [5, 1, 0, 8] * 9, [40, 17, 3, 200] * 9, 33, 0),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits,heads,kv,dim,page,new,lens,window,sinks", PAGED)
def test_paged_attention(t, bits, heads, kv, dim, page, new, lens, window, sinks):
    """Every split: with the hints of a real call, with none, and with hints that are too small."""
    g = _gen(dim + heads)
    used = [-(-n // page) for n in lens]
    width, pages = max(used) + 2, sum(used) + 2
    table = _tables(g, used, width, pages)
    cache = Cache(t, bits, kv, dim, page, pages, width)
    _fill(cache, g, table, lens)
    rows = sum(new) + 3
    q = _randn(g, cache.dt, rows, heads, dim)
    args = (cache, q, _ends(new), _i32(lens), _i32(table), heads, len(new), window, sinks)
    for hints in ({"max_new": max(new), "max_len": max(lens)}, {}, {"max_new": 1, "max_len": 1}, {"max_new": max(new), "max_len": 1 << 20}):
        o, _ = _run_paged(*args, **hints)
        _check_paged(cache, q, o, new, lens, table, window, sinks)


@pytest.mark.parametrize("bits", [8, 16])
def test_paged_attention_long(bits):
    """Thousands of keys, split over many work-groups and joined; twice the same bits."""
    g = _gen(5)
    lens, new = [9001, 4097, 1], [1, 2, 1]
    cache = Cache("bf16", bits, 2, 128, 16, 900, 600)
    table = _tables(g, [-(-n // 16) for n in lens], 600, 900)
    _fill(cache, g, table, lens)
    q = _randn(g, cache.dt, 4, 16, 128, scale=2.0)
    args = (cache, q, _ends(new), _i32(lens), _i32(table), 16, 3)
    o, n = _run_paged(*args, max_new=2, max_len=9001)
    assert n > 0
    _check_paged(cache, q, o, new, lens, table, 0, 0)
    for _ in range(3):
        assert torch.equal(_run_paged(*args, max_new=2, max_len=9001)[0].view(torch.int16), o.view(torch.int16))


def test_paged_attention_pages_without_tokens():
    """A page number outside the cache holds no key; a sequence of such pages alone gives zeros, and
    so does one of length zero or below, or with fewer tokens than new rows."""
    g = _gen(6)
    cache = Cache("f16", 8, 2, 64, 16, 8, 4)
    table = [[0, 1, 2, -1], [3, 4, 5, -1], [-1, 8, 1 << 30, -5], [6, -1, -1, -1], [7, -1, -1, -1]]
    lens = [48, 48, 48, 0, 1]
    _fill(cache, g, [table[0], table[1], [-1] * 4, table[3], table[4]], [48, 48, 0, 0, 1])
    q = _randn(g, cache.dt, 7, 4, 64)
    new = [1, 1, 1, 1, 3]
    holes = [table[0], [3, 9, 5, -1]] + table[2:]
    o, _ = _run_paged(cache, q, _ends(new), _i32(lens), _i32(holes), 4, 5)
    k, v = cache.rows(table[1], 48)
    keep = [i for i in range(48) if not 16 <= i < 32]
    r, av, err = _attend(q[1:2], k[keep], v[keep], torch.tensor([100], device="cuda"), True, 0, 0, 0.125)
    _close(o[1:2], r, av, err, cache.u, 32, v.abs().max())
    assert (o[2:6] == 0).all()  # no page, no token, two rows before the first token
    r, av, err = _attend(q[6:7], *cache.rows(table[4], 1), torch.tensor([0], device="cuda"), True, 0, 0, 0.125)
    _close(o[6:7], r, av, err, cache.u, 1, 8)
    o, _ = _run_paged(cache, q[:1], _ends([1]), _i32([-7]), _i32([table[0]]), 4, 1)
    assert (o == 0).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads", [1, 8])
def test_paged_attention_odd_values_reach_only_rows_that_see_them(bits, heads):
    """NaN (and with 16 bits infinities) among cached values: later tokens and tokens outside the window
    do not reach a row; keys that are NaN do not either."""
    g = _gen(7)
    cache = Cache("bf16", bits, 1, 64, 16, 12, 12)
    table = _tables(g, [10], 12, 12)
    n, m = 6, 150
    k, v = _randn(g, cache.dt, m, 1, 64), _randn(g, cache.dt, m, 1, 64)
    v[147, 0, 5] = math.nan
    v[120, 0, 50] = math.nan
    k[148, 0, 3] = math.nan
    if bits == 16:
        v[146, 0, 17], v[30, 0, 40], v[149, 0, 60] = math.inf, -math.inf, -math.inf
    for window, sinks in ((0, 0), (25, 0), (28, 31), (2, 0)):
        cache.append(k, v, None, None, _ends([m]), _i32([m]), _i32(table), 1)
        q = _randn(g, cache.dt, n, heads, 64)
        o, _ = _run_paged(cache, q, _ends([n]), _i32([m]), _i32(table), heads, 1, window, sinks)
        kk, vv = cache.rows(table[0], m)
        place = torch.arange(m - n, m, device="cuda")
        rows = [i for i in range(n) if not (m - n + i >= 148 and (not window or m - n + i - 148 < window))]  # key 148 unseen
        kk[148] = 0
        r, av, err = _attend(q[rows], kk, vv, place[rows], True, window, sinks, 0.125)
        _close(o[rows], r, av, err, cache.u, m, 4)
        hit = [i for i in range(n) if i not in rows]
        assert o[hit].isnan().all()


RAGGED = [  # heads, kv heads, dim, causal, window, sinks, lengths of queries, of keys (None: the same)
    (4, 4, 64, True, 0, 0, [1, 2, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 300], None),
    (4, 2, 128, True, 0, 0, [1, 200, 0, 513], None), (4, 1, 72, False, 0, 0, [400, 289, 1, 65], None),
    (3, 3, 32, False, 0, 0, [100, 7], None), (6, 2, 80, True, 0, 0, [150, 33], None), (2, 1, 96, False, 0, 0, [257], None),
    (2, 2, 256, True, 0, 0, [130, 64], None), (2, 1, 192, False, 0, 0, [129], None), (5, 5, 8, True, 0, 0, [70], None),
    (2, 1, 40, False, 0, 0, [70], None), (4, 2, 128, True, 64, 4, [400, 20, 129], None), (4, 2, 64, True, 1, 0, [200], None),
    (4, 2, 128, True, 100, 70, [513, 90], None), (4, 2, 128, False, 50, 9, [300, 64], None), (2, 2, 64, False, 1, 0, [130], None),
    (2, 1, 128, True, 200, 1, [700], None), (2, 1, 256, True, 33, 2, [257], None),
    (4, 2, 64, True, 0, 0, [5, 300, 64, 3, 0], [200, 64, 64, 0, 40]), (4, 2, 128, False, 0, 0, [5, 300, 7], [200, 64, 0]),
    (4, 2, 64, True, 40, 3, [5, 300, 64], [200, 64, 300]), (4, 2, 64, False, 40, 3, [5, 300, 64], [200, 64, 300]),
    # heads dealt to the XCDs in each way: one, two and seven for each, units in turn, and runs of work-groups
    (8, 1, 64, True, 0, 0, [300], None), (16, 4, 64, True, 0, 0, [700], None), (16, 2, 128, True, 90, 3, [300], [500]),
    (28, 2, 64, True, 0, 0, [200, 0, 129, 31], None), (16, 4, 64, True, 0, 0, [300, 7, 0, 129], None),
    (28, 4, 64, True, 0, 0, [300], None), (16, 4, 64, True, 0, 0, [300, 130, 5], None), (7, 1, 64, False, 0, 0, [129, 260], None),
    (6, 3, 64, True, 0, 0, [140] * 13, None),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv,dim,causal,window,sinks,nq,nk", RAGGED)
def test_attention(t, heads, kv, dim, causal, window, sinks, nq, nk):
    code, dt, u = TYPES[t]
    g = _gen(dim)
    nk = nq if nk is None else nk
    q = _randn(g, dt, sum(nq) + 5, heads, dim)
    k, v = _randn(g, dt, sum(nk) + 2, kv, dim), _randn(g, dt, sum(nk) + 2, kv, dim)
    k[sum(nk):], v[sum(nk):] = math.nan, math.nan
    scale = 1 / math.sqrt(dim)
    cq, ck = _ends(nq), _ends(nk)
    for max_q in (max(nq), 0, 1):
        o = torch.full_like(q, 5.0)
        d = ops.attention_desc(code, heads, kv, dim, scale, causal, window, sinks, max_q=max_q)
        ops.attention(d, _p(q), _p(k), _p(v), _p(cq), _p(ck), _p(o), len(nq), q.shape[0], k.shape[0], _stream())
        a, b = 0, 0
        for n, m in zip(nq, nk):
            place = torch.arange(m - n, m, device="cuda")
            r, av, err = _attend(q[a:a + n], k[b:b + m], v[b:b + m], place, causal, window, sinks, scale)
            _close(o[a:a + n], r, av, err, u, m, v[b:b + m].abs().max().double() if m else 0)
            a, b = a + n, b + m
        assert (o[a:] == 5.0).all()


def test_attention_strided_rows():
    """q, k, v cut from packed rows; output head by head; keys and values stored head by head."""
    code, dt, u = TYPES["f16"]
    g = _gen(11)
    n, heads, dim = 333, 3, 72
    rows = _randn(g, dt, n, 3 * heads * dim)
    q, k, v = (rows[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in range(3))
    st = (rows.stride(0), dim)
    kt, vt = (x.transpose(0, 1).contiguous() for x in (k, v))
    r, av, err = _attend(q, k, v, torch.arange(n, device="cuda"), False, 0, 0, 0.2)
    cu = _ends([n])
    for ks, kk, vv in ((st, k, v), ((dim, n * dim), kt, vt)):
        o = torch.full((heads, n, dim), 5.0, dtype=dt, device="cuda")
        d = ops.attention_desc(code, heads, heads, dim, 0.2, False, q=st, k=ks, v=ks, o=(dim, n * dim))
        ops.attention(d, _p(q), _p(kk), _p(vv), _p(cu), _p(cu), _p(o), 1, n, n, _stream())
        _close(o.transpose(0, 1), r, av, err, u, n, v.abs().max().double())


def test_attention_odd_values_reach_only_rows_that_see_them():
    for t, dim in (("f16", 64), ("bf16", 128)):
        code, dt, u = TYPES[t]
        g = _gen(12)
        n = 300
        cu = _ends([n])
        q, k, v = (_randn(g, dt, n, 2, dim) for _ in range(3))
        v[250, 0, 5], v[100, 1, 50], v[299, 0, 1], v[40, 0, 9] = math.nan, math.inf, -math.inf, math.nan
        k[298] = math.nan
        for causal, window, sinks in ((True, 0, 0), (True, 30, 0), (True, 20, 45), (False, 25, 3)):
            o = torch.empty_like(q)
            d = ops.attention_desc(code, 2, 2, dim, 0.1, causal, window, sinks)
            ops.attention(d, _p(q), _p(k), _p(v), _p(cu), _p(cu), _p(o), 1, n, n, _stream())
            i = torch.arange(n, device="cuda")
            hit = (i >= 298) if causal else (i - 298).abs() < window
            if causal and window:
                hit &= i - 298 < window
            kk = k.clone()
            kk[298] = 0
            r, av, err = _attend(q[~hit], kk, v, i[~hit], causal, window, sinks, 0.1)
            _close(o[~hit], r, av, err, u, n, 5)
            assert o[hit].isnan().all()


def test_attention_large_scores():
    """Scores of thousands: the running maximum keeps exponents in range."""
    code, dt, u = TYPES["bf16"]
    g = _gen(13)
    n = 260
    cu = _ends([n])
    q, k, v = (_randn(g, dt, n, 2, 64, scale=s) for s in (20.0, 20.0, 1.0))
    o = torch.empty_like(q)
    for scale in (1.0, -1.0, 0.0):
        d = ops.attention_desc(code, 2, 2, 64, scale)
        ops.attention(d, _p(q), _p(k), _p(v), _p(cu), _p(cu), _p(o), 1, n, n, _stream())
        r, av, err = _attend(q, k, v, torch.arange(n, device="cuda"), True, 0, 0, scale)
        # exponents of up to 2^14 here: their fp32 rounding is 2^-10 relative
        _close(o, r, av, err + 2.0 ** -9, u, n, 5)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("bits", [8, 16])
def test_prompt_then_tokens(bits):
    """A model's layer as a server runs it: a ragged prompt through rotation, append and ragged attention,
    then tokens one by one and drafted ones five at a time through rotation, append and paged
    attention, each against attention over everything so far."""
    code, dt, u = TYPES["bf16"]
    g = _gen(20)
    heads, kv, dim, page, sections = 8, 2, 128, 16, (24, 20, 20)
    prompt = [37, 1, 160]
    steps = [1, 1, 5, 1, 3, 1]
    total = [p + sum(steps) for p in prompt]
    cache = Cache("bf16", bits, kv, dim, page, 40, 14)
    table = _tables(g, [-(-n // page) for n in total], 14, 40)
    freq = _freq(64)
    lens = [0, 0, 0]
    for n, new in enumerate([prompt] + [[s] * 3 for s in steps]):
        rows = sum(new)
        qkv = _randn(g, dt, rows, (heads + 2 * kv) * dim)
        st = (qkv.stride(0), dim)
        q, k, v = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv) * dim], qkv[:, (heads + kv) * dim:]
        pos = torch.randint(0, 5000, (3, rows), generator=g, device="cuda", dtype=torch.int32)
        lens = [a + b for a, b in zip(lens, new)]
        cu, dl, tb = _ends(new), _i32(lens), _i32(table)
        cache.append(k, v, pos, freq, cu, dl, tb, 3, sections, False, True, st, st)
        qr = torch.empty((rows, heads, dim), dtype=dt, device="cuda")
        ops.rope(ops.rope_desc(code, heads, dim, sections, dealt=True, x=st, pos_axis=rows), _p(q), _p(pos), _p(freq), _p(qr), rows, _stream())
        if n == 0:  # the prompt attends to its own rows
            kr = torch.empty((rows, kv, dim), dtype=dt, device="cuda")
            ops.rope(ops.rope_desc(code, kv, dim, sections, dealt=True, x=st, pos_axis=rows), _p(k), _p(pos), _p(freq), _p(kr), rows, _stream())
            o = torch.empty_like(qr)
            ops.attention(ops.attention_desc(code, heads, kv, dim, 0.09, v=st, max_q=max(new)), _p(qr), _p(kr), _p(v), _p(cu), _p(cu), _p(o),
                          3, rows, rows, _stream())
            a = 0
            for m in new:
                r, av, err = _attend(qr[a:a + m], kr[a:a + m], v[a:a + m].unflatten(1, (kv, dim)), torch.arange(m, device="cuda"), True, 0, 0, 0.09)
                _close(o[a:a + m], r, av, err, u, m, 6)
                a += m
        o, _ = _run_paged(cache, qr, cu, dl, tb, heads, 3, max_new=max(new), max_len=max(lens), scale=0.09)
        _check_paged(cache, qr, o, new, lens, table, 0, 0, 0.09)
    assert lens == total


def test_graph_and_streams():
    """A decoding step captured into a graph and replayed with other lengths, positions and inputs, with
    eager work between; then on a side stream."""
    g = _gen(30)
    heads, kv, dim, page, batch = 8, 2, 128, 16, 4
    cache, plain = (Cache("f16", 8, kv, dim, page, 300, 80) for _ in range(2))
    start = [1000, 17, 500, 64]
    table = _tables(g, [-(-(n + 8) // page) for n in start], 80, 300)
    tb = _i32(table)
    state = g.get_state()
    _fill(cache, g, table, start)
    g.set_state(state)
    _fill(plain, g, table, start)
    rows = batch + 2
    k, v, q = (torch.zeros((rows, h, dim), dtype=torch.float16, device="cuda") for h in (kv, kv, heads))
    pos, lens, cu, freq = torch.zeros((1, rows), dtype=torch.int32, device="cuda"), _i32(start), _ends([1] * batch), _freq(64)
    qr, o = torch.zeros_like(q), torch.full_like(q, 5.0)
    rd = ops.rope_desc(ops.F16, heads, dim, (64,), pos_axis=rows)
    ad = ops.append_desc(cache.desc, (64,), pos_axis=rows)
    pd = ops.paged_attention_desc(cache.desc, heads, 0.09, max_new=1, max_len=80 * page)
    need = ops.paged_attention_workspace(pd, batch, rows)
    assert need > 0
    ws = [torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in range(2)]

    def step(c, out, w):
        s = _stream()
        ops.rope(rd, _p(q), _p(pos), _p(freq), _p(qr), rows, s)
        ops.kv_append(ad, _p(k), _p(v), _p(pos), _p(freq), _p(cu), _p(lens), _p(tb), _p(c.kc), _p(c.vc), _p(c.ks), _p(c.vs), batch, rows, s)
        ops.paged_attention(pd, _p(qr), _p(c.kc), _p(c.vc), _p(c.ks), _p(c.vs), _p(cu), _p(lens), _p(tb), _p(out), batch, rows, _p(w), need, s)

    def inputs(n):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        lens.copy_(_i32([m + n for m in start]))
        pos.copy_(torch.randint(0, 9000, pos.shape, generator=g, device="cuda", dtype=torch.int32))

    inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, o, ws[0])
    torch.cuda.current_stream().wait_stream(side)
    want = torch.full_like(q, 5.0)
    step(plain, want, ws[1])
    torch.cuda.synchronize()
    assert torch.equal(o, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, o, ws[0])
    for n in range(2, 7):
        inputs(n)
        graph.replay()
        step(plain, want, ws[1])
        torch.cuda.synchronize()
        assert torch.equal(o, want) and (o[batch:] == 5.0).all()
        assert torch.equal(cache.kc, plain.kc) and torch.equal(cache.vc, plain.vc)
        _check_paged(cache, qr[:batch], o[:batch], [1] * batch, [m + n for m in start], table, 0, 0, 0.09)


def test_offsets_past_32_bits():
    """Pages whose bytes lie past 2^32: the same codes and results as from pages at the start."""
    g = _gen(40)
    kv, dim, page, pages = 8, 128, 128, 36000  # 128 KB a page of keys: 4.7 GB, and as much of values
    desc = ops.cache_desc(ops.BF16, 8, kv, dim, page, pages, 4)
    nb, ns = ops.cache_bytes(desc)
    assert nb > 1 << 32
    kc, vc = (torch.empty(nb, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(ns // 4, device="cuda") for _ in range(2))
    n = 300
    k, v, q = (_randn(g, torch.bfloat16, n, h, dim) for h in (kv, kv, 16))
    cu, lens = _ends([n]), _i32([n])
    got = []
    for ids in ([0, 1, 2, -1], [pages - 1, pages - 3, pages - 2, -1]):
        table = _i32([ids])
        ops.kv_append(ops.append_desc(desc), _p(k), _p(v), None, None, _p(cu), _p(lens), _p(table), _p(kc), _p(vc), _p(ks), _p(vs), 1, n, _stream())
        d = ops.paged_attention_desc(desc, 16, 0.1, max_new=n, max_len=n)
        ws = torch.empty(max(16, ops.paged_attention_workspace(d, 1, n)), dtype=torch.uint8, device="cuda")
        o = torch.empty_like(q)
        ops.paged_attention(d, _p(q), _p(kc), _p(vc), _p(ks), _p(vs), _p(cu), _p(lens), _p(table), _p(o), 1, n, _p(ws), ws.numel(), _stream())
        at = torch.tensor(ids[:3], device="cuda")
        got.append([o, ks.reshape(pages, kv)[at], vs.reshape(pages, kv)[at]] + [torch.stack([c.reshape(pages, -1)[i] for i in ids[:3]]) for c in (kc, vc)])
    for a, b in zip(*got):
        # the last page's empty slots are whatever the memory held
        if a.dtype == torch.uint8:
            assert torch.equal(a[:2], b[:2])
        else:
            assert torch.equal(a, b)


def test_two_graphs_at_once():
    """Two captured calls with a workspace each, replayed on two streams at once, with a strided output."""
    g = _gen(41)
    heads, kv, dim, page = 16, 2, 128, 32
    lens, new = [5000, 3000], [1, 1]
    cache = Cache("bf16", 8, kv, dim, page, 300, 160)
    table = _tables(g, [-(-n // page) for n in lens], 160, 300)
    _fill(cache, g, table, lens)
    cu, dl, tb = _ends(new), _i32(lens), _i32(table)
    # output head by head
    d = ops.paged_attention_desc(cache.desc, heads, 0.09, o=(dim, 2 * dim), max_new=1, max_len=5000)
    need = ops.paged_attention_workspace(d, 2, 2)
    assert need > 0
    runs = []
    for _ in range(2):
        q, o = _randn(g, cache.dt, 2, heads, dim), torch.empty((heads, 2, dim), dtype=cache.dt, device="cuda")
        ws, s, graph = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            ops.paged_attention(d, _p(q), _p(cache.kc), _p(cache.vc), _p(cache.ks), _p(cache.vs), _p(cu), _p(dl), _p(tb), _p(o), 2, 2, _p(ws), need, _stream())
        runs.append((q, o, ws, s, graph))
    for _ in range(5):
        for q, o, ws, s, graph in runs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for q, o, ws, s, graph in runs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for q, o, ws, s, graph in runs:
            _check_paged(cache, q, o.transpose(0, 1), new, lens, table, 0, 0, 0.09)


def test_operands_that_are_not_on_the_device():
    x = torch.zeros((2, 1, 64), dtype=torch.float16)
    y = x.cuda()
    pos, freq = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), _freq(32)
    d = ops.rope_desc(ops.F16, 1, 64, (32,))
    with pytest.raises(RuntimeError, match="not device memory"):
        ops.rope(d, _p(x), _p(pos), _p(freq), _p(y), 2, _stream())
    ops.rope(d, _p(y), _p(pos), _p(freq), _p(y), 2, _stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_paged_attention_lengths_that_do_not_fit(bits, window, sinks):
    """Lengths below the number of new rows, of nothing, below 0 and behind the table's end; first rows
    that lie behind the rows there are: rows whose place is before the first key are zero."""
    g = _gen(8)
    page, width = 16, 4
    cache = Cache("bf16", bits, 2, 64, page, 20, width)
    new, lens = [4, 3, 2, 0, 1, 5], [2, 0, -5, 7, 1000, 64]
    stored = [min(max(n, 0), page * width) for n in lens]
    table = _tables(g, [-(-n // page) for n in stored], width, 20)
    _fill(cache, g, table, stored)
    rows = sum(new)
    q = _randn(g, cache.dt, rows, 8, 64)
    cu = _ends(new)
    cu[-1] += 1000
    for hints in ({}, {"max_new": 5, "max_len": 64}):
        o, _ = _run_paged(cache, q, cu, _i32(lens), _i32(table), 8, len(new), window, sinks, **hints)
        row = 0
        for b, (n, m, kept) in enumerate(zip(new, lens, stored)):
            k, v = cache.rows(table[b], kept)
            place = torch.arange(n, device="cuda") + max(m, 0) - n
            r, av, err = _attend(q[row:row + n], k, v, place, True, window, sinks, 0.125)
            _close(o[row:row + n], r, av, err, cache.u, kept, v.abs().max() if kept else 0)
            row += n
        assert (o[:2] == 0).all() and (o[4:9] == 0).all()


# ------------------------------------------------------------------ value scales far apart
def _fill_apart(cache, gen, table, lens, apart):
    """Pages whose value scales differ: page i of a sequence has values of zero (None), or 2^-apart[i] of
    ordinary ones; `apart` is repeated."""
    rows = sum(lens)
    k, v = (_randn(gen, cache.dt, rows, cache.heads, cache.dim) for _ in range(2))
    place = torch.cat([torch.arange(n, device="cuda") for n in lens])
    zero = torch.tensor([a is None for a in apart], device="cuda")[place // cache.page % len(apart)]
    v[zero] = 0
    cache.append(k, v, None, None, _ends(lens), _i32(lens), _i32(table), len(lens))
    vs = cache.vs.view(cache.pages, cache.heads)
    for ids in table:
        for i, at in enumerate(ids):
            if at >= 0 and apart[i % len(apart)]:
                vs[at] *= 2.0 ** -apart[i % len(apart)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (4, 1, 64, 32), (3, 3, 80, 16), (4, 2, 256, 64)])
@pytest.mark.parametrize("apart", [[0, None], [None] * 7 + [0], [0] + [None] * 7, [0, 12], [16, 0], [0, 20, 0, 24, None], [25, 0, 10]])
def test_paged_attention_value_scales_apart(t, heads, kv, dim, page, apart):
    """Keys of a page count with their weight however small the page's values are: pages of zeros before, between
    and behind ordinary ones, in a step, across steps and across parts; one new token and several.

    A small weight of fp16 is off by 2^-25 of the largest, in units of its page's codes: 448 times the scale
    at most, which is twice the page's largest value."""
    g = _gen(50 + dim)
    new, lens = [1, 3, 1, 1], [5 * page - 3, 130, 2, 300 * page - 7]
    used = [-(-n // page) for n in lens]
    table = _tables(g, used, max(used), sum(used))
    cache = Cache(t, 8, kv, dim, page, sum(used), max(used))
    _fill_apart(cache, g, table, lens, apart)
    q = _randn(g, cache.dt, sum(new), heads, dim, scale=0.5)
    q[0] = 0  # every key has the same weight
    for hints in ({"max_new": 3, "max_len": max(lens)}, {"max_new": 3, "max_len": 1}, {}):
        o, _ = _run_paged(cache, q, _ends(new), _i32(lens), _i32(table), heads, 4, **hints)
        row = 0
        for b, (n, m) in enumerate(zip(new, lens)):
            k, v = cache.rows(table[b], m)
            r, av, err = _attend(q[row:row + n], k, v, torch.arange(m - n, m, device="cuda"), True, 0, 0, 1 / math.sqrt(dim))
            _close(o[row:row + n], r, av, err, cache.u, m, 2 * v.abs().max())
            row += n


def test_paged_attention_value_scales_past_fp32():
    """bf16 values of 2^100 and more beside zeros: the pages' scales are further apart than the exponents
    of fp32 reach, and the zeros' keys count all the same."""
    g = _gen(60)
    lens, page = [133, 4000], 16
    used = [-(-n // page) for n in lens]
    table = _tables(g, used, max(used), sum(used))
    cache = Cache("bf16", 8, 2, 64, page, sum(used), max(used))
    _fill_apart(cache, g, table, lens, [-118, None, None, 0])
    q = _randn(g, cache.dt, 4, 4, 64, scale=0.5)
    for hints in ({"max_new": 2, "max_len": 4000}, {"max_new": 2, "max_len": 1}):
        o, _ = _run_paged(cache, q, _ends([2, 2]), _i32(lens), _i32(table), 4, 2, **hints)
        for b, m in enumerate(lens):
            k, v = cache.rows(table[b], m)
            r, av, err = _attend(q[2 * b:2 * b + 2], k, v, torch.arange(m - 2, m, device="cuda"), True, 0, 0, 0.125)
            _close(o[2 * b:2 * b + 2], r, av, err, cache.u, m, 2 * v.abs().max())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("scale", [0.0, 1e-35, -1e-30, -0.25])
def test_paged_attention_small_and_negative_scales(t, bits, scale):
    """A softmax scale of zero or nearly: the plain average of the values, over keys of zero too (whose pages
    have a scale of 2^-32), with a last page that is not full and a window that ends inside pages."""
    g = _gen(61)
    lens, new, page = [37, 150, 16], [1, 4, 2], 16
    used = [-(-n // page) for n in lens]
    table = _tables(g, used, 10, sum(used))
    cache = Cache(t, bits, 2, 64, page, sum(used), 10)
    rows = sum(lens)
    k, v = _randn(g, cache.dt, rows, 2, 64), _randn(g, cache.dt, rows, 2, 64)
    k[30:37], k[37 + 144:] = 0, 0
    cache.append(k, v, None, None, _ends(lens), _i32(lens), _i32(table), 3)
    q = _randn(g, cache.dt, sum(new) + 1, 4, 64)
    for window, sinks in ((0, 0), (21, 3)):
        o, _ = _run_paged(cache, q, _ends(new), _i32(lens), _i32(table), 4, 3, window, sinks, scale=scale)
        _check_paged(cache, q, o, new, lens, table, window, sinks, scale)


# ------------------------------------------------------------------ many small weights
def _few_and_many(gen, dt, n, kv, dim, low):
    """Queries, keys and values of which one key per head has a weight 2^low times the others', which vary by
    2^0.5 and less, and values of zero."""
    q = torch.zeros((1, kv, dim), device="cuda")
    q[..., 0], q[..., 1] = 1, 1
    k, v = torch.zeros((n, kv, dim), device="cuda"), _randn(gen, dt, n, kv, dim).abs() + 1
    k[:, :, 1] = torch.rand((n, kv), generator=gen, device="cuda") * 0.5
    k[n // 3, :, 0], k[n // 3, :, 1], v[n // 3] = low, 0, 0
    return q.to(dt), k.to(dt), v.to(dt)


def _small_weights_close(o, q, k, v, n, u):
    """fp16 weights from 2^-21 of the largest on are rounded by u of themselves, those below by 2^-32 of
    the largest; over 8-bit pages in units of the codes, 448 times the scale at most, which is twice the
    page's largest value."""
    r, av, err = _attend(q, k, v, torch.tensor([n - 1], device="cuda"), True, 0, 0, math.log(2))
    tol = u * r.abs() + u * av + 2 * (err + 2.0 ** -15) * av + n * 2.0 ** -31 * v.double().abs().max() + 2.0 ** -25
    assert ((o.double() - r).abs() <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("low", [14, 20, 25])
@pytest.mark.parametrize("n", [60, 16000])
def test_attention_many_small_weights(t, low, n):
    """Thousands of keys whose weights lie at and below fp16's lowest normal value, relative to one other's: what
    they add up to reaches the row."""
    code, dt, u = TYPES[t]
    q, k, v = _few_and_many(_gen(70), dt, n, 2, 64, low)
    o = torch.empty_like(q)
    cq, ck = _ends([1]), _ends([n])
    ops.attention(ops.attention_desc(code, 2, 2, 64, math.log(2)), _p(q), _p(k), _p(v), _p(cq), _p(ck), _p(o), 1, 1, n, _stream())
    _small_weights_close(o, q, k, v, n, u)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("low", [14, 20, 25])
@pytest.mark.parametrize("n", [60, 16000])
def test_paged_attention_many_small_weights(t, bits, low, n):
    cache = Cache(t, bits, 2, 64, 32, -(-n // 32), -(-n // 32))
    q, k, v = _few_and_many(_gen(71), cache.dt, n, 2, 64, low)
    table = [list(range(-(-n // 32)))]
    cache.append(k, v, None, None, _ends([n]), _i32([n]), _i32(table), 1)
    for hints in ({"max_new": 1, "max_len": n}, {"max_new": 1, "max_len": 1}):
        o, _ = _run_paged(cache, q, _ends([1]), _i32([n]), _i32(table), 2, 1, scale=math.log(2), **hints)
        _small_weights_close(o, q, *cache.rows(table[0], n), n, cache.u)


def test_paged_attention_lengths_near_the_largest():
    """Lengths of up to 2^31 - 1 over a table of a few pages: rows stand far behind the last key and see the
    first tokens alone, or with no window all there are."""
    g = _gen(9)
    cache = Cache("f16", 8, 2, 64, 16, 8, 8)
    table = [list(range(8))]
    _fill(cache, g, table, [128])
    q = _randn(g, cache.dt, 3, 4, 64)
    for n in ((1 << 31) - 1, (1 << 31) - 60, 1 << 30):
        for window, sinks in ((1, (1 << 31) - 1), (1 << 20, 70), ((1 << 31) - 1, 1), (5, 0), (0, 0)):
            o, _ = _run_paged(cache, q, _ends([3]), _i32([n]), _i32(table), 4, 1, window, sinks)
            k, v = cache.rows(table[0], 128)
            place = torch.arange(n - 3, n, device="cuda")
            r, av, err = _attend(q, k, v, place, True, window, sinks, 0.125)
            _close(o, r, av, err, cache.u, 128, v.abs().max())
