"""Attention with shared first tokens at sizes where one launch does not join all rows.

Tolerances are those of test_gpu_answers.py.
"""
import pytest
import torch

import test_gpu_seq as seq
from infvino_amd import ops
from test_gpu_answers import _space
from test_gpu_seq import Cache, _ends, _gen, _i32, _p, _randn, _stream

pytestmark = pytest.mark.gpu


def test_rows_of_more_than_one_join():
    """2^22 rows of 256 channels and a few more: the first and the last sequences against the definition, those in between
    against the first, whose queries they repeat (each is off by u |o| + u sum w |v| and little more, u = 2^-8 and sums around 1)."""
    g = _gen(81)
    heads, dim, page, lens = 64, 256, 128, 150
    batch = (1 << 16) + 3
    cache = Cache("bf16", 8, 1, dim, page, 3, 2)
    seq._fill(cache, g, [[2, 0]], [lens])
    some = _randn(g, cache.dt, 64, heads, dim)
    q = some.repeat(batch // 64 + 1, 1, 1)[:batch].contiguous()
    o = torch.full((batch + 1, heads, dim), 5.0, dtype=cache.dt, device="cuda")
    d = ops.prefix_attention_desc(cache.desc, heads, dim ** -0.5, max_new=1, max_len=lens, max_shared=page)
    need = ops.prefix_attention_workspace(d, batch, 1, batch)
    space, cu, length, table = _space(need), _ends([1] * batch), _i32([lens] * batch), _i32([[2, 0]]).repeat(batch, 1)
    member, shared = _i32([0, batch]), _i32([page])
    ops.prefix_attention(d, _p(q), _p(cache.kc), _p(cache.vc), _p(cache.ks), _p(cache.vs), _p(cu), _p(length), _p(table), _p(member), _p(shared), _p(o),
                         batch, 1, batch, _p(space), need, _stream())
    for part in (slice(0, 64), slice(batch - 64, batch)):
        seq._check_paged(cache, q[part], o[part], [1] * 64, [lens] * 64, [[2, 0]] * 64, 0, 0)
    for i in range(64, batch - 64, 64):
        assert torch.allclose(o[i:i + 64].float(), o[:64].float(), rtol=2 ** -6, atol=2 ** -6)
    assert (o[batch] == 5.0).all()
