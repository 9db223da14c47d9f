"""Attention with shared first tokens where many rows of up to 64 channels read a long prefix 128 at a time.  That kernel is taken
for 512 rows of a group and more where the tables hold 16384 tokens and more and max_shared says as many, so the tables
here are that wide; the shared tokens themselves may be few, since max_shared only steers the split.

Tolerances are those of test_gpu_answers.py.
"""
import math

import pytest
import torch

import test_gpu_seq as seq
from infvino_amd import ops
from test_gpu_answers import FEW, LONG, Shared, _space
from test_gpu_seq import TYPES, _ends, _gen, _i32, _p, _randn, _stream

pytestmark = pytest.mark.gpu


class Wide(Shared):
    """Tables of 16384 tokens."""

    def __init__(self, gen, t, bits, kv, dim, page, *rest, **kw):
        super().__init__(gen, t, bits, kv, dim, page, *rest, **kw)
        width = max(16384 // page, self.cache.width)
        self.table = [row + [-1] * (width - len(row)) for row in self.table]
        self.cache.width = self.cache.desc.table_width = width

    def run(self, q, heads, hints=LONG, groups=None, **kw):
        """The workspace shows that the call is split for 128 rows at a time: 768 work-groups over shared keys, not 256 of 32 rows."""
        n, c = len(self.sizes) if groups is None else groups, self.cache
        if n:
            rows, steps = -(-q.shape[0] // n) * heads // c.heads, c.width * c.page // 64

            def parts(want):
                return -(-steps // -(-steps // min(max(want, 1), steps, 256)))
            many, wide = parts(768 // (n * c.heads * -(-rows // 128))), parts(-(-256 // (n * c.heads * -(-rows // 32))))
            d = ops.prefix_attention_desc(c.desc, heads, 1.0, max_new=hints[0], max_len=hints[1], max_shared=hints[2])
            assert ops.prefix_attention_workspace(d, self.batch, n, q.shape[0]) == (many + 1) * q.shape[0] * heads * (c.dim + 2) * 4 and many != wide
        return super().run(q, heads, hints=hints, groups=groups, **kw)


ROWS = [  # heads, kv heads, dim, page, sizes, shared, new, own
    (64, 2, 64, 64, [20], [1000], [1] * 20, [1 + 3 * i for i in range(20)]),  # 640 rows: five full tiles
    (64, 1, 48, 16, [18, 16], [129, 65], [1] * 34, [1 + i % 5 for i in range(34)]),  # two groups, channels behind the head's end
    (64, 1, 16, 128, [33], [1500], [1] * 33, [1] * 33),
    (32, 1, 32, 32, [17, 21, 16], [700, 63, 3000], [1] * 54, [1 + i % 7 for i in range(54)]),  # one group has no whole step
    (28, 4, 64, 16, [80], [333], [1] * 80, [1 + i for i in range(80)]),  # 7 heads a key head
    (64, 8, 64, 128, [20], [300], [1 + i % 7 for i in range(20)], [8 + i for i in range(20)]),  # drafted tokens
    (16, 1, 64, 32, [3], [1000], [40, 1, 30], [40, 7, 90]),  # 1136 rows, pieces of prompts
    (64, 1, 64, 16, [9], [64], [1] * 9, [1] * 9),  # one step
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads,kv,dim,page,sizes,shared,new,own", ROWS)
def test_many_rows(t, bits, heads, kv, dim, page, sizes, shared, new, own):
    g = _gen(dim + len(own))
    s = Wide(g, t, bits, kv, dim, page, sizes, shared, new, own)
    q = _randn(g, s.cache.dt, sum(new) + 3, heads, dim)
    s.check(q, s.run(q, heads, hints=LONG))


@pytest.mark.parametrize("bits", [8, 16])
def test_many_rows_behind_a_prefix_that_is_long(bits):
    g = _gen(71)
    s = Wide(g, "bf16", bits, 1, 64, 128, [9], [16500], [1] * 9, [1 + i for i in range(9)])
    q = _randn(g, torch.bfloat16, 9, 64, 64)
    s.check(q, s.run(q, 64, hints=FEW))


def _check_rows(s, got, q, scale):
    """As sequences of the pages that are there; infinities reach the rows that see them."""
    row, page = 0, s.cache.page
    for b, (n, m) in enumerate(zip(s.new, s.lens)):
        ids = s.table[b][:-(-m // page)]
        ks, vs = s.cache.rows([max(0, min(i, s.cache.pages - 1)) for i in ids], m)
        ok = torch.tensor([0 <= i < s.cache.pages for i in ids], device="cuda").repeat_interleave(page)[:m]
        place = torch.arange(m - n, m, device="cuda")
        for i in range(n):
            see = ok & (torch.arange(m, device="cuda") <= place[i])
            r, av, err = seq._attend(q[row:row + 1], ks[see], vs[see], torch.tensor([int(see.sum())], device="cuda"), True, 0, 0, scale)
            seq._close(got[row:row + 1], r, av, err, s.cache.u, m, vs[see].abs().nan_to_num(0, 0, 0).max() if see.any() else 0)
            row += 1


@pytest.mark.parametrize("dim", [48, 64])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("scale", [0.25, -0.25, 0.0, 1e-30])
def test_many_rows_pages_that_hold_nothing(bits, dim, scale):
    """Among the shared ones, whatever their bytes are; softmax scales of each sign."""
    g = _gen(72)
    s = Wide(g, "f16", bits, 1, dim, 16, [12], [400], [1] * 12, [1 + 9 * i for i in range(12)])
    for i in range(12):
        s.table[i][3] = -1
        s.table[i][4] = s.cache.pages
        s.table[i][17] = 1 << 30
    q = _randn(g, torch.float16, 12, 64, dim)
    _check_rows(s, s.run(q, 64, hints=LONG, scale=scale), q, scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 16])
def test_many_rows_groups_and_lengths_of_every_kind(t, bits):
    """Sequences of no group; ones that end before the shared tokens do; empty groups; no group at all; a page of nothing in a
    whole step of them."""
    g = _gen(73)
    s = Wide(g, t, bits, 1, 64, 16, [12, 10], [300, 200], [1] * 22 + [2, 1], [1 + i for i in range(22)] + [90, 1], alone=2)
    q = _randn(g, s.cache.dt, sum(s.new), 64, 64)
    for kw in ({}, {"groups": 0}, {"groups": 1, "member": _i32([0, 12]), "shared": _i32([288])}, {"groups": 1, "member": _i32([12, 22]), "shared": _i32([192])}):
        s.check(q, s.run(q, 64, hints=LONG, **kw))
    short = list(s.lens)
    s.lens[5] = 40  # within the shared tokens, which are read by each alone then
    s.check(q, s.run(q, 64, hints=LONG))
    s.lens = short
    for row in s.table[:12]:
        row[4:12] = [-1] * 8  # two whole steps
    _check_rows(s, s.run(q, 64, hints=LONG), q, 0.125)


@pytest.mark.parametrize("bits", [8, 16])
def test_many_rows_odd_values(bits):
    """An infinity among the shared values reaches every row, one among a sequence's own that sequence alone, and a NaN
    among the shared keys every row's every channel."""
    g = _gen(74)
    s = Wide(g, "f16", bits, 1, 64, 32, [10], [320], [1] * 10, [40] * 10)
    q = _randn(g, torch.float16, 10, 64, 64)
    e = 16 if bits == 8 else 8
    dt = torch.uint8 if bits == 8 else torch.float16
    vc = s.cache.vc.view(dt).view(s.cache.pages, 1, 32 // e, 64, e)
    kc = s.cache.kc.view(dt).view(s.cache.pages, 1, 8, 64 // e, 4, e)
    odd = 0x7f if bits == 8 else math.nan
    own, shared = s.table[4][320 // 32], s.table[0][2]
    was = vc[own, 0, 0, 5, 2].clone(), vc[shared, 0, 1, 9, 3].clone(), kc[shared, 0, 2, 1, 1, 0].clone()
    vc[own, 0, 0, 5, 2] = odd
    bad = ~s.run(q, 64, hints=LONG).isfinite()
    assert bad[4, :, 5].all() and int(bad.sum()) == 64
    vc[own, 0, 0, 5, 2] = was[0]
    vc[shared, 0, 1, 9, 3] = odd
    bad = ~s.run(q, 64, hints=LONG).isfinite()
    assert bad[:, :, 9].all() and int(bad.sum()) == 640
    vc[shared, 0, 1, 9, 3] = was[1]
    kc[shared, 0, 2, 1, 1, 0] = odd
    assert not s.run(q, 64, hints=LONG).isfinite().any()
    kc[shared, 0, 2, 1, 1, 0] = was[2]
    s.check(q, s.run(q, 64, hints=LONG))


@pytest.mark.parametrize("heads,dim,rows,long", [(64, 64, 64, True), (64, 64, 64, False), (64, 128, 64, False), (8, 64, 2, False), (8, 128, 2, False)])
def test_shared_pages_past_32_bits(heads, dim, rows, long):
    """Each way that shared keys are taken (128, 32 and 16 rows at a time) gives the same bits for the same pages at the front of
    the cache and past 2^32 bytes of it."""
    g = _gen(75)
    kv, page = (8, 128)
    bits = 16 if dim == 64 else 8
    pages = 36000
    desc = ops.cache_desc(ops.BF16, bits, kv, dim, page, pages, 16384 // page)
    nb, ns = ops.cache_bytes(desc)
    assert nb > 1 << 32
    kc, vc = (torch.empty(nb, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(ns // 4, device="cuda") if bits == 8 else None for _ in range(2))
    k, v = (_randn(g, torch.bfloat16, 300, kv, dim) for _ in range(2))
    q = _randn(g, torch.bfloat16, rows, heads, dim)
    got = []
    for first in (3, pages - 9):
        table = [first + 4, first, first + 7] + [-1] * (16384 // page - 3)
        one, seq_lens, ids = _ends([300]), _i32([300]), _i32(table)
        ops.kv_append(ops.append_desc(desc), _p(k), _p(v), None, None, _p(one), _p(seq_lens), _p(ids), _p(kc), _p(vc), _p(ks), _p(vs), 1, 300, _stream())
        o = torch.empty_like(q)
        d = ops.prefix_attention_desc(desc, heads, 0.09, max_new=1, max_shared=16384 if long else 256)
        n = ops.prefix_attention_workspace(d, rows, 1, rows)
        space = _space(n)
        cu, lens, tables, member, shared = _ends([1] * rows), _i32([300] * rows), _i32([table] * rows), _i32([0, rows]), _i32([256])
        ops.prefix_attention(d, _p(q), _p(kc), _p(vc), _p(ks), _p(vs), _p(cu), _p(lens), _p(tables), _p(member), _p(shared), _p(o), rows, 1, rows, _p(space),
                             n, _stream())
        got.append(o)
    assert got[0].isfinite().all() and torch.equal(got[0], got[1])


def test_the_same_call_gives_the_same_bits():
    g = _gen(76)
    for bits in (8, 16):
        for cls, heads, kv, dim, hints in ((Wide, 64, 1, 64, LONG), (Shared, 64, 1, 64, FEW), (Shared, 64, 1, 128, FEW), (Shared, 8, 2, 128, FEW)):
            s = cls(g, "bf16", bits, kv, dim, 16, [12], [400], [1] * 12, [1 + 9 * i for i in range(12)])
            q = _randn(g, torch.bfloat16, 12, heads, dim)
            first = s.run(q, heads, hints=hints)
            for _ in range(5):
                assert torch.equal(first, s.run(q, heads, hints=hints))
