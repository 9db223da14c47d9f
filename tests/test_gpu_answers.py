"""Operators of a program that answers one prompt many times, on the GPU against their definitions in 64 bits: attention over
a cache with shared first pages, linear attention with decays, sampling, and a run of them together.

Tolerances (u = half a step of the type relative to the value: 2^-11 fp16, 2^-8 bf16):
  shared prefix  those of attention over a paged cache (test_gpu_seq.py): the join of parts adds a few roundings of 2^-24
  linear         with B = scale (sum over s <= t of decay |q| . |k_s| |v_s|, and decay |q| |S|) for an output:
                 u |o| for its rounding, u B for scores rounded to the type, 2^-16 B for states in two parts of 16 bits
                 (2^-18), decays (2^-22 each of few), and fp32 sums of up to 64 + 256 terms (2^-15.6 at worst), and
                 2^-25 for fp16's subnormal values.
                 States, with A = sum of decay |k| |v| and decay |S|: values with decays are held to 2^-22 in fp16, 2^-24 in
                 bf16, products summed in fp32 over n tokens: (n + 16) 2^-23 A, decays to 2^-22 for each token and
                 chunk: n 2^-22 A; fp16's parts are off by 2^-39 of the largest value with its decay where they are subnormal:
                 2^-38 max decay |v| sum |k|
  sampling       whole numbers, equal
"""
import math

import numpy as np
import pytest
import torch

import test_gpu_seq as seq
from infvino_amd import ops
from test_gpu_seq import TYPES, Cache, _ends, _gen, _i32, _p, _randn, _stream

pytestmark = pytest.mark.gpu


def _space(n):
    """A workspace whose contents do not matter: NaN, -1."""
    return torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------ shared prefixes
class Shared:
    """Groups of sequences that share their first pages: sizes, declared shared tokens, new and own tokens of each sequence."""

    def __init__(self, gen, t, bits, kv, dim, page, sizes, shared, new, own, alone=0):
        self.batch, self.sizes, self.new = sum(sizes) + alone, sizes, new
        held = [s // page * page for s, n in zip(shared, sizes) for _ in range(n)] + [0] * alone
        self.lens = [h + o for h, o in zip(held, own)]
        used = [max(1, -(-n // page)) for n in self.lens]
        width = max(used + [s // page for s in shared]) + 1
        pages = sum(s // page for s in shared) + sum(used) + 2
        order = torch.randperm(pages, generator=gen, device="cuda").tolist()
        self.cache = Cache(t, bits, kv, dim, page, pages, width)
        self.table, b, first = [], 0, []
        for n, s in list(zip(sizes, shared)) + [(1, 0)] * alone:
            head = [order.pop() for _ in range(s // page)]
            first.append(head + [-1] * (width - len(head)))
            for _ in range(n):
                tail = [order.pop() for _ in range(max(0, used[b] - len(head)))]
                self.table.append(head + tail + [-1] * (width - len(head) - len(tail)))
                b += 1
        starts = [s // page * page for s in shared]
        if sum(starts):
            seq._fill(self.cache, gen, first[:len(sizes)], starts)
        mine = [max(0, n - h) for n, h in zip(self.lens, held)]
        if sum(mine):
            k, v = (_randn(gen, self.cache.dt, sum(mine), kv, dim) for _ in range(2))
            self.cache.append(k, v, None, None, _ends(mine), _i32(self.lens), _i32(self.table), self.batch)
        self.member, self.shared = _i32([0] + list(np.cumsum(sizes))), _i32(shared)

    def run(self, q, heads, o=None, hints=(0, 0, 0), groups=None, space=None, scale=None, member=None, shared=None):
        c = self.cache
        o = torch.full_like(q, 5.0) if o is None else o
        groups = len(self.sizes) if groups is None else groups
        d = ops.prefix_attention_desc(c.desc, heads, 1 / math.sqrt(c.dim) if scale is None else scale, q=q.stride()[:2], o=o.stride()[:2],
                                      max_new=hints[0], max_len=hints[1], max_shared=hints[2])
        n = ops.prefix_attention_workspace(d, self.batch, groups, q.shape[0])
        space = _space(n) if space is None else space
        cu, lens, table = _ends(self.new), _i32(self.lens), _i32(self.table)  # alive until the call has them
        ops.prefix_attention(d, _p(q), _p(c.kc), _p(c.vc), _p(c.ks), _p(c.vs), _p(cu), _p(lens), _p(table),
                             _p(self.member if member is None else member), _p(self.shared if shared is None else shared), _p(o), self.batch, groups,
                             q.shape[0], _p(space), n, _stream())
        return o

    def check(self, q, o, scale=None):
        seq._check_paged(self.cache, q, o, self.new, self.lens, self.table, 0, 0, scale)


FEW, MANY = (0, 0, 0), (0, 0, 8192)  # hints; the latter is more than these tables hold, and is cut to that
PREFIX = [  # bits, heads, kv heads, dim, page, sizes, shared, new, own, hints
    (8, 8, 2, 128, 16, [4], [200], [1] * 4, [1, 2, 17, 70], FEW),
    (8, 8, 2, 128, 16, [1], [64], [1], [1], FEW),
    (8, 4, 4, 64, 32, [3, 2], [131, 0], [1, 1, 2, 1, 3], [1, 40, 100, 1, 3], FEW),
    (8, 28, 4, 80, 64, [2, 3, 1], [63, 640, 64], [1] * 6, [5, 1, 64, 65, 300, 2], FEW),
    (8, 8, 1, 256, 128, [5], [1300], [1, 0, 2, 0, 1], [1, 3, 2, 0, 129], FEW),
    (8, 6, 2, 16, 16, [9], [77], [1] * 9, list(range(1, 10)), FEW),
    (8, 8, 2, 144, 16, [20], [330], [3] * 20, [3 + 7 * i for i in range(20)], FEW),
    (16, 8, 2, 128, 16, [4], [200], [1] * 4, [1, 2, 17, 70], FEW),
    (16, 28, 4, 96, 64, [2, 3, 1], [63, 640, 64], [1] * 6, [5, 1, 64, 65, 300, 2], FEW),
    (16, 4, 4, 64, 32, [3, 2], [131, 0], [1, 1, 2, 1, 3], [1, 40, 100, 1, 3], FEW),
    (16, 8, 1, 256, 128, [5], [1300], [1, 0, 2, 0, 1], [1, 3, 2, 0, 129], FEW),
    (8, 8, 2, 128, 16, [70], [260], [2] * 70, [2 + i % 9 for i in range(70)], (2, 300, 256)),
    (8, 16, 1, 64, 16, [3], [1000], [40, 1, 30], [40, 7, 90], FEW),
    # many rows
    (8, 32, 1, 128, 16, [17], [330], [1] * 17, [1 + i for i in range(17)], MANY),
    (8, 64, 2, 64, 64, [20], [1000], [1] * 20, [1 + 3 * i for i in range(20)], MANY),
    (8, 32, 1, 80, 32, [33], [200], [1] * 33, [1] * 33, MANY),
    (8, 64, 1, 256, 128, [9], [520], [1] * 9, [2] * 9, MANY),
    (8, 32, 1, 48, 16, [18, 16], [129, 65], [1] * 34, [1 + i % 5 for i in range(34)], MANY),
    (8, 32, 1, 208, 16, [16, 17], [64, 700], [1] * 33, [1 + i % 5 for i in range(33)], MANY),
    (16, 32, 1, 128, 16, [17], [330], [1] * 17, [1 + i for i in range(17)], MANY),
    (16, 64, 2, 64, 64, [20], [1000], [1] * 20, [1 + 3 * i for i in range(20)], MANY),
    (16, 32, 1, 80, 32, [33], [200], [1] * 33, [1] * 33, MANY),
    (16, 64, 1, 256, 128, [9], [520], [1] * 9, [2] * 9, MANY),
    (16, 32, 1, 208, 16, [16, 17], [64, 700], [1] * 33, [1 + i % 5 for i in range(33)], MANY),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits,heads,kv,dim,page,sizes,shared,new,own,hints", PREFIX)
def test_prefix_attention(t, bits, heads, kv, dim, page, sizes, shared, new, own, hints):
    g = _gen(dim + len(own))
    s = Shared(g, t, bits, kv, dim, page, sizes, shared, new, own)
    q = _randn(g, s.cache.dt, sum(new) + 3, heads, dim)
    s.check(q, s.run(q, heads, hints=hints))


@pytest.mark.parametrize("hints,heads,kv", [(FEW, 8, 2), (MANY, 64, 1)])
@pytest.mark.parametrize("bits", [8, 16])
def test_prefix_attention_groups_and_lengths_of_every_kind(bits, hints, heads, kv):
    """Sequences of no group; one that ends before the shared tokens do, which then are read by each alone; no group at all;
    pages that hold nothing among the shared ones and the others; tokens declared beyond the tables."""
    g = _gen(7)
    s = Shared(g, "bf16", bits, kv, 64, 16, [12, 4], [300, 200], [1] * 16 + [2, 1], [1 + i for i in range(16)] + [90, 1], alone=2)
    q = _randn(g, torch.bfloat16, sum(s.new), heads, 64)
    s.check(q, s.run(q, heads, hints=hints))
    s.check(q, s.run(q, heads, hints=hints, member=_i32([0, 12, 16]), shared=_i32([300, 1 << 30])[:2].clamp(max=192)))
    s.check(q, s.run(q, heads, hints=hints, groups=0))
    s.check(q, s.run(q, heads, hints=hints, groups=3, member=_i32([0, 5, 5, 12]), shared=_i32([100, 50, 288])))
    s.check(q, s.run(q, heads, hints=hints, groups=1, member=_i32([3, 3]), shared=_i32([288])))
    short = list(s.lens)
    s.lens[5], s.lens[14] = 40, 70  # within the shared tokens
    s.check(q, s.run(q, heads, hints=hints))
    s.lens = short
    for row in s.table[:12]:
        row[3], row[17] = -1, s.cache.pages  # shared
    s.table[13][12] = -7
    table, s.table = s.table, [list(r) for r in s.table]
    got = s.run(q, heads, hints=hints)
    # as sequences of the pages that are there
    row = 0
    k, v = s.cache.values()
    for b, (n, m) in enumerate(zip(s.new, s.lens)):
        ids = table[b][:-(-m // 16)]
        ks, vs = s.cache.rows([max(0, min(i, s.cache.pages - 1)) for i in ids], m)
        ok = torch.tensor([0 <= i < s.cache.pages for i in ids], device="cuda").repeat_interleave(16)[:m]
        place = torch.arange(m - n, m, device="cuda")
        for i in range(n):
            see = ok & (torch.arange(m, device="cuda") <= place[i])
            r, av, err = seq._attend(q[row:row + 1], ks[see], vs[see], torch.tensor([int(see.sum())], device="cuda"), True, 0, 0, 0.125)
            seq._close(got[row:row + 1], r, av, err, s.cache.u, m, vs[see].abs().max() if see.any() else 0)
            row += 1


LONG = (0, 0, 16384)  # as MANY: rows are taken 128 at a time where tables hold as much (test_gpu_prefix_rows.py)
PREFIX_LONG = [
    (8, 64, 2, 64, 64, [20], [1000], [1] * 20, [1 + 3 * i for i in range(20)], LONG),
    (8, 64, 1, 48, 16, [18, 16], [129, 65], [1] * 34, [1 + i % 5 for i in range(34)], LONG),
    (16, 64, 2, 64, 64, [20], [1000], [1] * 20, [1 + 3 * i for i in range(20)], LONG),
    (16, 64, 1, 48, 16, [18, 16], [129, 65], [1] * 34, [1 + i % 5 for i in range(34)], LONG),
    (8, 64, 1, 16, 128, [33], [16500], [1] * 33, [1] * 33, FEW),
    (8, 8, 2, 128, 16, [30], [2100], [1] * 30, [1 + i for i in range(30)], FEW),  # 120 rows: 32 at a time
    (16, 6, 1, 112, 32, [17, 16], [700, 65], [1] * 33, [1 + i for i in range(33)], FEW),
    # more groups, and more sequences, than lanes look at together
    (8, 4, 2, 64, 16, [2] * 70, [64 + 16 * i for i in range(70)], [1 + i % 2 for i in range(140)], [2 + i % 40 for i in range(140)], FEW),
    (16, 4, 2, 128, 16, [100, 33], [200, 70], [1] * 133, [1 + i % 40 for i in range(133)], FEW),
    (8, 4, 2, 64, 16, [63, 65], [200, 70], [1] * 128, [1 + i % 40 for i in range(128)], FEW),
    (8, 4, 2, 64, 16, [1] * 63, [64 + 16 * i for i in range(63)], [1] * 63, [2] * 63, FEW),
    (8, 4, 2, 64, 16, [1] * 64, [64 + 16 * i for i in range(64)], [1] * 64, [2] * 64, FEW),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits,heads,kv,dim,page,sizes,shared,new,own,hints", PREFIX_LONG)
def test_prefix_attention_long(t, bits, heads, kv, dim, page, sizes, shared, new, own, hints):
    g = _gen(dim + len(own))
    s = Shared(g, t, bits, kv, dim, page, sizes, shared, new, own)
    q = _randn(g, s.cache.dt, sum(new) + 3, heads, dim)
    s.check(q, s.run(q, heads, hints=hints))


@pytest.mark.parametrize("hints,dim", [(LONG, 64), (FEW, 64), (FEW, 128)])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("scale", [0.25, -0.25, 0.0])
def test_prefix_attention_pages_that_hold_nothing(bits, hints, dim, scale):
    """Among the shared ones, whatever their bytes are; softmax scales of each sign."""
    g = _gen(31)
    s = Shared(g, "f16", bits, 1, dim, 16, [12], [400], [1] * 12, [1 + 9 * i for i in range(12)])
    for i in range(12):
        s.table[i][3] = -1
        s.table[i][4] = s.cache.pages
        s.table[i][17] = 1 << 30
    q = _randn(g, torch.float16, 12, 64, dim)
    got = s.run(q, 64, hints=hints, scale=scale)
    for b, m in enumerate(s.lens):
        ids = s.table[b][:-(-m // 16)]
        ks, vs = s.cache.rows([max(0, min(i, s.cache.pages - 1)) for i in ids], m)
        ok = torch.tensor([0 <= i < s.cache.pages for i in ids], device="cuda").repeat_interleave(16)[:m]
        r, av, err = seq._attend(q[b:b + 1], ks[ok], vs[ok], torch.tensor([int(ok.sum())], device="cuda"), True, 0, 0, scale)
        seq._close(got[b:b + 1], r, av, err, s.cache.u, m, vs[ok].abs().max())


@pytest.mark.parametrize("hints,heads", [(FEW, 8), (MANY, 64)])
@pytest.mark.parametrize("bits", [8, 16])
def test_prefix_attention_odd_values_stay_with_their_rows(bits, hints, heads):
    """An infinity among one sequence's own values reaches that sequence alone; behind a sequence's last token anything may
    stand; strided rows."""
    g = _gen(11)
    s = Shared(g, "f16", bits, 1, 64, 32, [10], [320], [1] * 10, [40] * 10)
    wide = _randn(g, torch.float16, 10, heads + 2, 80)
    q = wide[:, 1:heads + 1, 8:72]
    page = s.table[4][320 // 32]
    e = 16 if bits == 8 else 8
    vc = s.cache.vc.view(torch.uint8 if bits == 8 else torch.float16).view(s.cache.pages, 1, 32 // e, 64, e)
    odd = 0x7f if bits == 8 else math.inf
    vc[page, 0, 0, 5, 2] = odd
    out = torch.full((10, heads, 72), 5.0, dtype=torch.float16, device="cuda")
    o = s.run(q, heads, o=out[:, :, :64], hints=hints)
    assert (out[:, :, 64:] == 5.0).all()
    bad = ~o.isfinite()
    assert bad[4, :, 5].all() and int(bad.sum()) == heads
    vc[page, 0, 0, 5, 2] = 0
    s.check(q, s.run(q, heads, hints=hints))


def test_prefix_attention_is_paged_attention():
    """Scales of 0 and below, and the same sequences without sharing, agree to the tolerance of either."""
    g = _gen(12)
    s = Shared(g, "bf16", 8, 2, 128, 16, [6], [640], [1] * 6, [3, 90, 1, 16, 17, 200])
    q = _randn(g, torch.bfloat16, 6, 8, 128)
    for scale in (0.0, -0.1, 1e-30, 0.3):
        s.check(q, s.run(q, 8, scale=scale), scale)


def test_prefix_attention_past_32_bits():
    """Shared pages whose bytes lie past 2^32 in both kinds of split."""
    g = _gen(13)
    kv, dim, page, pages = 8, 128, 128, 36000
    desc = ops.cache_desc(ops.BF16, 8, kv, dim, page, pages, 5)
    nb, ns = ops.cache_bytes(desc)
    kc, vc = (torch.empty(nb, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(ns // 4, device="cuda") for _ in range(2))
    k, v = (_randn(g, torch.bfloat16, 300, kv, dim) for _ in range(2))
    q = _randn(g, torch.bfloat16, 64, 64, dim)
    for hints in (FEW, MANY):
        got = []
        for first in (3, pages - 9):
            table = [first + 4, first, first + 7, -1, -1]
            one, seq_lens, rows = _ends([300]), _i32([300]), _i32(table)
            ops.kv_append(ops.append_desc(desc), _p(k), _p(v), None, None, _p(one), _p(seq_lens), _p(rows), _p(kc), _p(vc), _p(ks), _p(vs), 1, 300, _stream())
            o = torch.empty_like(q)
            d = ops.prefix_attention_desc(desc, 64, 0.09, max_new=1, max_len=300, max_shared=hints[2])
            n = ops.prefix_attention_workspace(d, 64, 1, 64)
            space = _space(n)
            cu, lens, tables, member, shared = _ends([1] * 64), _i32([300] * 64), _i32([table] * 64), _i32([0, 64]), _i32([256])
            ops.prefix_attention(d, _p(q), _p(kc), _p(vc), _p(ks), _p(vs), _p(cu), _p(lens), _p(tables), _p(member), _p(shared), _p(o), 64, 1, 64, _p(space),
                                 n, _stream())
            got.append(o)
        assert torch.equal(got[0], got[1])


# ------------------------------------------------------------------ linear attention
def _linear_ref(q, k, v, g, state, scale):
    """One sequence: q, k [n][heads][dk], v [n][heads][dv], g [n][heads], state [heads][dk][dv] in 64 bits.
    (o, its B, last state, its A, sum |k| max decay |v|)."""
    n = q.shape[0]
    q, k, v, state = (x.double() for x in (q, k, v, state))
    b = g.double().clamp(min=-1e4).cumsum(0).t()  # [heads][n]
    q, k, v = (x.transpose(0, 1) for x in (q, k, v))
    if n == 0:
        return v.transpose(0, 1), v.transpose(0, 1), state, state.abs(), torch.zeros_like(state[..., :1])
    late = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    w = torch.exp((b[:, :, None] - b[:, None]).masked_fill(~late, -math.inf))
    o = scale * ((w * (q @ k.transpose(1, 2))) @ v + torch.exp(b)[..., None] * (q @ state))
    big = abs(scale) * ((w * (q.abs() @ k.abs().transpose(1, 2))) @ v.abs() + torch.exp(b)[..., None] * (q.abs() @ state.abs()))
    left = torch.exp(b[:, -1:] - b)[..., None]
    s = torch.exp(b[:, -1])[:, None, None] * state + (left * k).transpose(1, 2) @ v
    a = torch.exp(b[:, -1])[:, None, None] * state.abs() + (left * k.abs()).transpose(1, 2) @ v.abs()
    return o.transpose(0, 1), big.transpose(0, 1), s, a, k.abs().sum(1)[..., None] * (left * v.abs()).amax(1)[:, None]


class Linear:
    def __init__(self, gen, t, heads, key_heads, dk, dv, lens, pad=2, decay="each", slots=None):
        self.code, self.dt, self.u = TYPES[t]
        self.heads, self.kh, self.dk, self.dv, self.lens = heads, key_heads, dk, dv, lens
        n = sum(lens) + pad
        self.q, self.k = _randn(gen, self.dt, n, key_heads, dk), _randn(gen, self.dt, n, key_heads, dk, scale=dk ** -0.5)
        self.v = _randn(gen, self.dt, n, heads, dv)
        slow = torch.exp(torch.linspace(math.log(1e-3), math.log(3.0), heads, device="cuda"))
        self.g = -slow * torch.rand((n, heads), generator=gen, device="cuda") if decay == "each" else -slow
        self.slots = 2 * len(lens) if slots is None else slots
        self.state = torch.randn((self.slots, heads, dk, dv), generator=gen, device="cuda")
        self.start, self.to = list(range(len(lens))), [len(lens) + i for i in range(len(lens))]

    def run(self, scale=0.125, max_new=0, state=None, o=None, to=True):
        o = torch.full((self.q.shape[0], self.heads, self.dv), 5.0, dtype=self.dt, device="cuda") if o is None else o
        state = self.state.clone() if state is None else state
        gs = (self.g.stride(0), self.g.stride(1)) if self.g.dim() == 2 else (0, self.g.stride(0))
        d = ops.linear_attention_desc(self.code, self.heads, self.kh, self.dk, self.dv, scale, self.slots, q=self.q.stride()[:2], k=self.k.stride()[:2],
                                      v=self.v.stride()[:2], o=o.stride()[:2], g=gs, max_new=max_new)
        n = ops.linear_attention_workspace(d, len(self.lens), self.q.shape[0])
        space = _space(n)
        start, to, cu = None if self.start is None else _i32(self.start), _i32(self.to) if to else None, _ends(self.lens)
        ops.linear_attention(d, _p(self.q), _p(self.k), _p(self.v), _p(self.g), _p(cu), _p(start), _p(to), _p(state), _p(o),
                             len(self.lens), self.q.shape[0], _p(space), n, _stream())
        return o, state, n

    def check(self, o, state, scale=0.125):
        want, row, rep = self.state.double(), 0, self.heads // self.kh
        wrote = set()
        for b, n in enumerate(self.lens):
            part = slice(row, row + n)
            at = -1 if self.start is None else self.start[b]
            first = self.state[at] if 0 <= at < self.slots else torch.zeros_like(self.state[0])
            g = self.g[part] if self.g.dim() == 2 else self.g.expand(n, -1)
            r, big, s, a, keys = _linear_ref(self.q[part].repeat_interleave(rep, 1), self.k[part].repeat_interleave(rep, 1), self.v[part], g, first, scale)
            tol = self.u * r.abs() + (self.u + 2.0 ** -16) * big + 2.0 ** -25
            bad = ~((o[part].double() - r).abs() <= tol)
            if bad.any():
                at = tuple(bad.nonzero()[0].tolist())
                print("sequence", b, "of", n, "off at", at, float(o[part][at]), float(r[at]), "tolerance", float(tol[at]), "count", int(bad.sum()))
            assert not bad.any()
            if 0 <= self.to[b] < self.slots:
                wrote.add(self.to[b])
                tol = (3 * n + 16) * 2.0 ** -23 * a + (2.0 ** -38 * keys if self.dt == torch.float16 else 0) + 1e-37
                bad = ~((state[self.to[b]].double() - s).abs() <= tol)
                if bad.any():
                    at = tuple(bad.nonzero()[0].tolist())
                    print("state", b, "of", n, "off at", at, float(state[self.to[b]][at]), float(s[at]), "tolerance", float(tol[at]), "count", int(bad.sum()))
                assert not bad.any()
            row += n
        assert (o[row:] == 5.0).all(), "rows of no sequence changed"
        for i in range(self.slots):
            if i not in wrote:
                assert torch.equal(state[i], self.state[i])


LINEAR = [  # heads, key heads, key dim, dim, lens
    (1, 1, 16, 16, [1]), (2, 1, 64, 64, [64]), (4, 2, 128, 128, [65, 0, 1, 63, 2]), (3, 3, 48, 80, [130, 17]), (2, 2, 256, 32, [70, 5, 128]),
    (2, 1, 96, 256, [200]), (1, 1, 128, 144, [129, 64]), (6, 2, 32, 96, [3, 300, 40]), (2, 2, 176, 208, [100, 33]), (8, 4, 128, 64, [1] * 40),
    (5, 5, 64, 128, [i % 7 for i in range(70)]), (2, 1, 256, 256, [90]), (4, 1, 112, 112, [191, 192, 193]),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("heads,kh,dk,dv,lens", LINEAR)
def test_linear_attention(t, heads, kh, dk, dv, lens, max_new):
    """In chunks (0: lengths unknown), and token by token."""
    x = Linear(_gen(dk + dv), t, heads, kh, dk, dv, lens, decay="each" if len(lens) != 2 else "head")
    o, state, _ = x.run(max_new=max_new)
    x.check(o, state)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kh,dk,dv,lens", [(2, 1, 128, 128, [1500, 40, 700]), (1, 1, 64, 80, [2100]), (2, 2, 256, 64, [900, 1025]), (1, 1, 48, 208, [1, 1600, 0])])
def test_linear_attention_in_segments(t, heads, kh, dk, dv, lens):
    """Long sequences by several work-groups; each sequence's state in its own slot, in place."""
    x = Linear(_gen(dk), t, heads, kh, dk, dv, lens)
    x.to = x.start
    o, state, need = x.run()
    assert need > 0
    x.check(o, state)


@pytest.mark.parametrize("max_new", [0, 1])
def test_linear_attention_slots(max_new):
    """Many sequences begin with one state; with none; leave theirs in place, or nowhere."""
    x = Linear(_gen(3), "bf16", 3, 1, 64, 48, [5, 0, 70, 1, 33, 0], slots=9)
    x.start, x.to = [2, 2, 2, -1, 9, 2], [4, 5, -1, 7, 8, 1 << 30]
    o, state, _ = x.run(max_new=max_new)
    x.check(o, state)
    x.start, x.to = [0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5]
    o, state, _ = x.run(max_new=max_new)
    x.check(o, state)
    x.start, x.to = None, [-1] * 6
    for to in (True, False):
        o, state, _ = x.run(max_new=max_new, to=to)
        x.check(o, state)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("kind", ["none", "all", "some", "strong", "grow", "slow"])
def test_linear_attention_decays(t, max_new, kind):
    """Decays of 1; that forget everything at every token or at some; of 2^-300; above 1; of 1 - 2^-13."""
    x = Linear(_gen(5), t, 2, 1, 64, 64, [100, 64, 3])
    x.g = {"none": torch.zeros_like(x.g), "all": torch.full_like(x.g, -math.inf), "some": torch.where(x.g < -0.5, -math.inf, 0.1 * x.g),
           "strong": torch.full_like(x.g, -208.0), "grow": 0.02 * torch.ones_like(x.g), "slow": torch.full_like(x.g, -2.0 ** -13)}[kind]
    o, state, _ = x.run(max_new=max_new)
    x.check(o, state)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
def test_linear_attention_sizes_of_values(t, max_new):
    """Scores past fp16's largest value and far below its smallest, states of 2^40 and 2^-40, small values."""
    for sq, sk, sv, ss in ((200.0, 200.0, 1e-3, 1.0), (1e-3, 1e-3, 1.0, 1.0), (1.0, 1.0, 1e-3, 1e-3), (1e-4, 1.0, 1.0, 2.0 ** 40), (100.0, 0.1, 1e-2, 2.0 ** -40)):
        x = Linear(_gen(6), t, 2, 2, 128, 64, [90, 5])
        x.q, x.k, x.v, x.state = (x.q.float() * sq).to(x.dt), (x.k.float() * sk).to(x.dt), (x.v.float() * sv).to(x.dt), x.state * ss
        scale = min(1.0, 1.0 / (sq * sk * sv * 100), 100.0 / (sq * ss))
        o, state, _ = x.run(scale=scale, max_new=max_new)
        x.check(o, state, scale=scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("what", ["q", "k", "v", "state"])
@pytest.mark.parametrize("odd", [math.inf, math.nan])
def test_linear_attention_odd_values_reach_no_earlier_row(t, max_new, what, odd):
    x = Linear(_gen(8), t, 2, 2, 64, 96, [70, 20, 130])
    clean, _, _ = x.run(max_new=max_new)
    at, head, ch = 70 + 20 + 75, 1, 33
    if what == "state":
        x.state[2, head, 7, ch] = odd
    else:
        getattr(x, what)[at, head, ch] = odd
    o, state, _ = x.run(max_new=max_new)
    first = {"q": at, "k": at, "v": at, "state": 90}[what]
    last = at + 1 if what == "q" else 220
    same = torch.ones_like(o, dtype=torch.bool)
    channels = slice(ch, ch + 1) if what in ("v", "state") else slice(None)
    same[first:last, head, channels] = False
    assert torch.equal(o[same], clean[same])
    assert not o[first:last, head, channels].isfinite().any()
    assert state[:, 0].isfinite().all() and state[3:5].isfinite().all()


@pytest.mark.parametrize("max_new", [0, 1])
def test_linear_attention_strides(max_new):
    """q, k, v cut from packed rows, outputs into wider ones, decays of a transposed buffer."""
    g = _gen(9)
    x = Linear(g, "f16", 4, 2, 64, 96, [70, 3])
    rows = _randn(g, torch.float16, 75, 2 * 64 + 2 * 64 + 4 * 104 + 8)
    x.q, x.k = rows[:, :128].unflatten(1, (2, 64)), (rows[:, 128:256] * 0.125).unflatten(1, (2, 64))
    x.v = rows[:, 256:256 + 416].unflatten(1, (4, 104))[:, :, 8:]
    x.g = x.g.t().contiguous().t()
    wide = torch.full((75, 5, 112), 5.0, dtype=torch.float16, device="cuda")
    o, state, _ = x.run(max_new=max_new, o=wide[:, 1:, 8:104])
    x.check(o, state)
    assert (wide[:, 0] == 5.0).all() and (wide[:, :, :8] == 5.0).all() and (wide[:, :, 104:] == 5.0).all()


def test_linear_attention_prompt_then_tokens():
    """A prompt at once, or cut anywhere and continued from the state, by either kernel."""
    x = Linear(_gen(10), "bf16", 4, 2, 128, 128, [150], pad=0)
    o, state, _ = x.run()
    for cut in (1, 64, 100, 149):
        y = Linear(_gen(10), "bf16", 4, 2, 128, 128, [150], pad=0)
        parts, s = [], y.state.clone()
        for lo, hi, slot_in, slot_out, hint in ((0, cut, 0, 1, 0), (cut, 150, 1, 1, 1)):
            z = Linear(_gen(1), "bf16", 4, 2, 128, 128, [hi - lo], pad=0)
            z.q, z.k, z.v, z.g = (a[lo:hi].contiguous() for a in (y.q, y.k, y.v, y.g))
            z.start, z.to = [slot_in], [slot_out]
            got, s, _ = z.run(max_new=hint, state=s)
            parts.append(got)
        y.check(torch.cat(parts), s)


# ------------------------------------------------------------------ sampling
def _weights(x, t):
    """Weights in whole multiples of 2^-44 (Python integers fit: at most 2^63)."""
    x = x.double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    with np.errstate(all="ignore"):
        z = np.where(x == top, 0.0, (x - top) * (1.4426950408889634 / t))
        z[~(x > -np.inf)] = -np.inf
        w = np.where(z > -45, np.maximum(np.rint(np.exp2(np.maximum(z, -60)) * 2.0 ** 44), 1), 0)
    return x, w.astype(np.uint64)


def _draw(x, t=1.0, k=0, p=1.0, m=0.0, u=0.5):
    x0 = x.float()
    if not (x0 > -math.inf).any():
        return -1
    if not t > 0:
        y = torch.nan_to_num(x0, nan=-math.inf, posinf=math.inf, neginf=-math.inf).cpu().numpy()
        return int(np.argmax(y))
    x, w = _weights(x0, t)
    order = np.lexsort((np.arange(len(x)), -x))
    ws = w[order]
    count = int((ws > 0).sum())
    if 0 < k < len(x):
        count = min(count, k)
    if p < 1:
        sums = np.cumsum(ws[:count])
        need = max(1, math.ceil(max(float(np.float32(p)), 0.0) * float(sums[-1])))
        count = min(count, int(np.searchsorted(sums, np.uint64(need))) + 1)
    kept = np.zeros(len(x), bool)
    kept[order[:count]] = True
    if m > 0:
        kept &= w >= np.uint64(max(1, math.ceil(min(float(np.float32(m)), 1.0) * 2.0 ** 44)))
    sums = np.cumsum(np.where(kept, w, 0).astype(np.uint64))
    total = int(sums[-1])
    goal = 0 if not u > 0 else total - 1 if u >= 1 else min(int(float(np.float32(u)) * float(total)), total - 1)
    return int(np.searchsorted(sums, np.uint64(goal), side="right"))


def _sample(x, t=None, k=None, p=None, m=None, u=None, type=None):
    rows, vocab = x.shape
    kind = {torch.float16: ops.F16, torch.bfloat16: ops.BF16, torch.float32: ops.F32}[x.dtype]
    f = lambda v, dt=torch.float32: None if v is None else torch.tensor(v, dtype=dt, device="cuda")  # noqa: E731
    t, k, p, m, u = f(t), f(k, torch.int32), f(p), f(m), f(u)
    out = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    d = ops.sample_desc(kind, vocab, row=x.stride(0))
    n = ops.sample_workspace(d, rows)
    space = _space(n)
    ops.sample(d, _p(x), _p(t), _p(k), _p(p), _p(m), _p(u), _p(out), rows, _p(space), n, _stream())
    return out.tolist()


DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 4096, 4097, 8191, 8192, 8193, 12289, 50021, 131073, 1 << 19])
def test_sample(dt, vocab):
    g = _gen(vocab)
    rows = 24 if vocab < 60000 else 12
    x = (torch.randn((rows, vocab + 3), generator=g, device="cuda") * 3).to(dt)[:, 1:vocab + 1]  # 2-byte alignment
    rng = np.random.default_rng(vocab)
    u = rng.random(rows).astype(np.float32).tolist()
    pick = lambda values: [values[i] for i in rng.integers(0, len(values), rows)]  # noqa: E731
    for t, k, p, m in ((None, None, None, None), ([0.7] * rows, pick([0, 1, 5, 50, 3000]), None, None), (pick([0.3, 1.0, 2.0]), None, pick([0.1, 0.5, 0.9, 0.999, 1.0]), None),
                       (pick([0.5, 1.5, 0.0]), pick([0, 2, 20, 1000]), pick([0.3, 0.95, 1.0]), pick([0.0, 0.01, 0.3, 1.0])), (None, None, None, pick([0.05, 0.5]))):
        got = _sample(x, t, k, p, m, u)
        want = [_draw(x[i], *(d if a is None else a[i] for a, d in ((t, 1.0), (k, 0), (p, 1.0), (m, 0.0))), u[i]) for i in range(rows)]
        assert got == want, (t, k, p, m)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("vocab", [5, 9000, 70000])
def test_sample_ties(dt, vocab):
    """Equal logits: in the order of their indexes, however many."""
    us = [0.0, 0.1, 0.25, 0.5, 0.75, 0.999, 1.0 - 2.0 ** -24]
    x = torch.full((len(us), vocab), 1.5, dtype=dt, device="cuda")
    assert _sample(x, u=us) == [min(int(float(np.float32(u)) * vocab), vocab - 1) for u in us]
    for k in (1, 2, 3, vocab - 1):
        assert _sample(x, k=[k] * len(us), u=us) == [min(int(float(np.float32(u)) * k), k - 1) for u in us]
    half = math.ceil(0.5 * vocab)
    assert _sample(x, p=[0.5] * len(us), u=us) == [min(int(float(np.float32(u)) * half), half - 1) for u in us]
    assert _sample(x, t=[0.0] * len(us), u=us) == [0] * len(us)
    x[:, vocab // 2:] = 0.5  # two values, ties on both sides of the cut
    for k, p in ((vocab // 2 + 2, 1.0), (0, 0.9), (vocab // 3, 0.7)):
        got = _sample(x, k=[k] * len(us), p=[p] * len(us), u=us)
        assert got == [_draw(x[i], 1.0, k, p, 0.0, u) for i, u in enumerate(us)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("vocab", [64, 8193, 40000])
def test_sample_odd_rows(dt, vocab):
    """Forbidden tokens as -infinity, as the type's lowest value, NaN; rows without a token; infinities; odd numbers."""
    g = _gen(vocab)
    low = torch.finfo(dt).min
    base = torch.randn((1, vocab), generator=g, device="cuda").to(dt)
    rows = [torch.full_like(base, -math.inf), torch.full_like(base, math.nan), torch.full_like(base, low)]
    for v in (-math.inf, low, math.nan):
        y = torch.full_like(base, v)
        y[0, [3, vocab // 2, vocab - 1]] = base[0, :3]
        rows.append(y)
    y = base.clone()
    y[0, [5, vocab - 2]] = math.inf
    rows.append(y)
    y = base.clone()
    y[0, 7], y[0, 9] = -0.0, 0.0
    rows += [y, base * 0, -base.abs() * 0]
    x = torch.cat(rows)
    n = len(rows)
    for t in (1.0, 0.0, -1.0, math.nan, math.inf, 1e-30, 1e-42, 1e30):
        for k, p, m, u in ((0, 1.0, 0.0, 0.3), (2, 0.9, 0.0, 0.9), (0, 0.0, 0.0, 0.99), (0, -1.0, 0.0, 0.5), (-5, math.nan, math.nan, 0.6), (0, 2.0, 5.0, 0.4), (vocab, 1.0, 1.0, 1.0),
                           (1, 1.0, 0.0, math.nan), (0, 0.5, 0.0, -1.0), (3, 0.99, 1e-9, 7.0)):
            got = _sample(x, [t] * n, [k] * n, [p] * n, [m] * n, [u] * n)
            want = [_draw(x[i], t, k, 1.0 if math.isnan(p) else p, 0.0 if math.isnan(m) else m, u) for i in range(n)]
            assert got == want, (t, k, p, m, u)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_sample_flat_rows(dt):
    """More tokens where the cut lies than are listed."""
    g = _gen(2)
    x = (torch.randn((6, 60000), generator=g, device="cuda") * 0.01).to(dt)
    u = [0.01, 0.3, 0.5, 0.77, 0.9, 0.99]
    for k, p, m in ((30000, 1.0, 0.0), (0, 0.5, 0.0), (50000, 0.4, 0.0), (0, 0.9, 0.985), (25000, 0.999, 0.0)):
        got = _sample(x, k=[k] * 6, p=[p] * 6, m=[m] * 6, u=u)
        assert got == [_draw(x[i], 1.0, k, p, m, u[i]) for i in range(6)], (k, p, m)


def test_sample_many_rows():
    """More rows than the chip has work-groups for parts of them; each row its own filters."""
    g = _gen(4)
    rows, vocab = 2500, 9001
    x = (torch.randn((rows, vocab), generator=g, device="cuda") * 2).bfloat16()
    rng = np.random.default_rng(1)
    t, u = (0.5 + rng.random(rows)).astype(np.float32).tolist(), rng.random(rows).astype(np.float32).tolist()
    k, p = rng.integers(-1, 60, rows).tolist(), rng.random(rows).astype(np.float32).tolist()
    got = _sample(x, t, k, p, None, u)
    pick = list(range(0, rows, 83))
    assert [got[i] for i in pick] == [_draw(x[i], t[i], k[i], p[i], 0.0, u[i]) for i in pick]


# ------------------------------------------------------------------ together
def test_answers_to_one_prompt():
    """A prompt's keys cached once and its linear state kept once; five answers that share both, token after token, in eager
    calls and as a graph that is replayed with the program's own work in between; every step against 64 bits."""
    g = _gen(20)
    n, prompt, steps, heads, kv, dim, page, vocab = 5, 150, 4, 8, 2, 64, 16, 9000
    dt = torch.bfloat16
    s = Shared(g, "bf16", 8, kv, dim, page, [n], [prompt], [1] * n, [prompt % page] * n)
    width = s.cache.width
    # each answer has the prompt's last, partial page of its own and one more
    lin = Linear(g, "bf16", heads, heads, dim, dim, [prompt], pad=0, slots=n + 1)
    lin.start, lin.to = [-1], [n]
    o, state, _ = lin.run()
    lin.check(o, state)
    names = ("q", "k", "v", "g", "lens", "start", "logits", "u")
    buf = {"q": torch.zeros((n, heads, dim), dtype=dt, device="cuda"), "k": torch.zeros((n, kv, dim), dtype=dt, device="cuda"),
           "v": torch.zeros((n, kv, dim), dtype=dt, device="cuda"), "lv": torch.zeros((n, heads, dim), dtype=dt, device="cuda"),
           "g": torch.zeros((n, heads), device="cuda"), "lens": _i32([prompt] * n), "start": _i32([n] * n), "u": torch.zeros(n, device="cuda")}
    weight = _randn(g, dt, heads * dim, vocab, scale=0.05)
    outs = {"o": torch.full((n, heads, dim), 5.0, dtype=dt, device="cuda"), "lo": torch.full((n, heads, dim), 5.0, dtype=dt, device="cuda"),
            "logits": torch.zeros((n, vocab), dtype=dt, device="cuda"), "token": torch.zeros(n, dtype=torch.int32, device="cuda")}
    fixed = {"cu": _ends([1] * n), "to": _i32(list(range(n))), "table": _i32(s.table), "t": torch.full((n,), 0.8, device="cuda"),
             "k": _i32([0, 5, 40, 0, 1]), "p": torch.tensor([0.9, 1.0, 0.7, 1.0, 1.0], device="cuda")}
    c = s.cache
    pd = ops.prefix_attention_desc(c.desc, heads, 0.125, max_new=1, max_len=prompt + steps, max_shared=prompt)
    ld = ops.linear_attention_desc(ops.BF16, heads, heads, dim, dim, 0.125, n + 1, max_new=1)
    sd = ops.sample_desc(ops.BF16, vocab)
    need = [ops.prefix_attention_workspace(pd, n, 1, n), ops.linear_attention_workspace(ld, n, n), ops.sample_workspace(sd, n)]
    space = [_space(x) for x in need]

    def step(state):
        c.append(buf["k"], buf["v"], None, None, fixed["cu"], buf["lens"], fixed["table"], n)
        ops.prefix_attention(pd, _p(buf["q"]), _p(c.kc), _p(c.vc), _p(c.ks), _p(c.vs), _p(fixed["cu"]), _p(buf["lens"]), _p(fixed["table"]), _p(s.member),
                             _p(s.shared), _p(outs["o"]), n, 1, n, _p(space[0]), need[0], _stream())
        ops.linear_attention(ld, _p(outs["o"]), _p(buf["q"]), _p(buf["lv"]), _p(buf["g"]), _p(fixed["cu"]), _p(buf["start"]), _p(fixed["to"]), _p(state),
                             _p(outs["lo"]), n, n, _p(space[1]), need[1], _stream())
        torch.matmul(outs["lo"].reshape(n, -1), weight, out=outs["logits"])
        ops.sample(sd, _p(outs["logits"]), _p(fixed["t"]), _p(fixed["k"]), _p(fixed["p"]), None, _p(buf["u"]), _p(outs["token"]), n, _p(space[2]), need[2], _stream())

    def inputs(i):
        for name in ("q", "k", "v", "lv"):
            buf[name].copy_(_randn(g, dt, *buf[name].shape))
        buf["g"].copy_(-torch.rand((n, heads), generator=g, device="cuda"))
        buf["u"].copy_(torch.rand(n, generator=g, device="cuda"))
        buf["lens"].fill_(prompt + i + 1)
        buf["start"].copy_(_i32([n] * n) if i == 0 else fixed["to"])

    def check(i, before, after):
        s.lens = [prompt + i + 1] * n
        s.check(buf["q"], outs["o"], 0.125)
        x = Linear(_gen(0), "bf16", heads, heads, dim, dim, [1] * n, pad=0, slots=n + 1)
        x.q, x.k, x.v, x.g, x.state, x.start, x.to = outs["o"], buf["q"], buf["lv"], buf["g"], before, buf["start"].tolist(), list(range(n))
        x.check(outs["lo"], after)
        want = [_draw(outs["logits"][b], float(fixed["t"][b]), int(fixed["k"][b]), float(fixed["p"][b]), 0.0, float(buf["u"][b])) for b in range(n)]
        assert outs["token"].tolist() == want

    live = state.clone()
    inputs(0)
    before = live.clone()
    step(live)
    check(0, before, live)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    inputs(1)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(live)
    for i in range(1, steps):
        inputs(i)
        before = live.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(i, before, live)
    assert names


def test_two_calls_at_once():
    """Each operator on two streams at once, and as two graphs, with a workspace each."""
    g = _gen(21)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    s = Shared(g, "f16", 8, 2, 64, 16, [9], [600], [1] * 9, [30 + 9 * i for i in range(9)])
    q = [_randn(g, torch.float16, 9, 8, 64) for _ in range(2)]
    lins = [Linear(_gen(22 + i), "f16", 1, 1, 128, 128, [1500, 300]) for i in range(2)]
    x = [(torch.randn((3, 30000), generator=g, device="cuda") * 2) for _ in range(2)]
    u, p = torch.tensor([0.2, 0.6, 0.9], device="cuda"), torch.tensor([0.8, 0.9, 0.99], device="cuda")
    c = s.cache
    pd = ops.prefix_attention_desc(c.desc, 8, 0.125, max_new=1, max_len=700, max_shared=600)
    sd = ops.sample_desc(ops.F32, 30000)
    ends, lens, table = _ends(s.new), _i32(s.lens), _i32(s.table)
    runs = []
    for i, stream in enumerate((a, b)):
        y = lins[i]
        ld = ops.linear_attention_desc(ops.F16, 1, 1, 128, 128, 0.125, y.slots)
        o, lo, token = torch.empty_like(q[i]), torch.empty_like(y.v), torch.empty(3, dtype=torch.int32, device="cuda")
        need = [ops.prefix_attention_workspace(pd, 9, 1, 9), ops.linear_attention_workspace(ld, 2, y.q.shape[0]), ops.sample_workspace(sd, 3)]
        space = [_space(z) for z in need]
        state, cu, start, to = y.state.clone(), _ends(y.lens), _i32(y.start), _i32(y.to)

        def go(i=i, y=y, ld=ld, o=o, lo=lo, token=token, need=need, space=space, state=state, cu=cu, start=start, to=to):
            ops.prefix_attention(pd, _p(q[i]), _p(c.kc), _p(c.vc), _p(c.ks), _p(c.vs), _p(ends), _p(lens), _p(table), _p(s.member), _p(s.shared),
                                 _p(o), 9, 1, 9, _p(space[0]), need[0], _stream())
            ops.linear_attention(ld, _p(y.q), _p(y.k), _p(y.v), _p(y.g), _p(cu), _p(start), _p(to), _p(state), _p(lo), 2, y.q.shape[0], _p(space[1]),
                                 need[1], _stream())
            ops.sample(sd, _p(x[i]), None, None, _p(p), None, _p(u), _p(token), 3, _p(space[2]), need[2], _stream())
        runs.append((stream, go, o, lo, state, token, torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()

    def check():
        torch.cuda.synchronize()
        for i, (_, _, o, lo, state, token, _) in enumerate(runs):
            s.check(q[i], o, 0.125)
            n = sum(lins[i].lens)
            full = torch.full_like(lo, 5.0)
            full[:n] = lo[:n]
            lins[i].check(full, state)
            assert token.tolist() == [_draw(x[i][r], 1.0, 0, float(p[r]), 0.0, float(u[r])) for r in range(3)]

    for _ in range(3):
        for stream, go, *_ in runs:
            with torch.cuda.stream(stream):
                go()
        check()
    for stream, go, *_, graph in runs:
        with torch.cuda.graph(graph, stream=stream):
            go()
    for _ in range(4):
        for _, _, o, lo, state, token, _ in runs:
            o.fill_(3.0)
            token.fill_(-5)
        torch.cuda.synchronize()
        for stream, *_, graph in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        check()


def test_operands_that_are_not_on_the_device():
    x, u, token = torch.zeros((1, 10)), torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="not device memory"):
        ops.sample(ops.sample_desc(ops.F32, 10), _p(x), None, None, None, None, _p(u), _p(token), 1, None, 0, _stream())
    y = Linear(_gen(0), "f16", 1, 1, 16, 16, [2])
    y.q = y.q.cpu()
    with pytest.raises(RuntimeError, match="not device memory"):
        y.run()
    torch.cuda.synchronize()
