"""Linear attention at the ends of what its header allows: decays above 1, states and values far apart in size.

Tolerances are those of test_gpu_answers.py, which hold for any decays: bounds are formed with the decays that the reference uses.
"""
import math

import pytest
import torch

from test_gpu_answers import Linear
from test_gpu_seq import TYPES, _gen

pytestmark = pytest.mark.gpu


def _scale(x, most=1000.0):
    """A power of two by which the largest output, in 64 bits, comes to less than `most` (fp16 holds up to 65504)."""
    big, row, rep = 0.0, 0, x.heads // x.kh
    for b, n in enumerate(x.lens):
        q, k, v, g = (y[row:row + n].double() for y in (x.q, x.k, x.v, x.g))
        s = x.state[x.start[b]].double().clone()
        for t in range(n):
            s = torch.exp(g[t])[:, None, None] * s + k[t].repeat_interleave(rep, 0)[:, :, None] * v[t][:, None]
            big = max(big, float((q[t].abs().repeat_interleave(rep, 0)[:, None] @ s.abs()).max()))
        row += n
    return 2.0 ** math.floor(math.log2(most / big))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("up", [0.1, 0.2, 0.5, 0.6])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 96), (256, 32)])
def test_growing_decays(t, max_new, up, dk, dv):
    """Factors above 1 at every token: up to e^60 over a sequence, values past fp16's range long before a chunk's end."""
    x = Linear(_gen(dk + dv), t, 2, 1, dk, dv, [100, 64, 3])
    x.v = x.v * 1000 if up == 0.1 else x.v
    x.g = torch.full_like(x.g, up)
    scale = _scale(x)
    o, state, _ = x.run(scale=scale, max_new=max_new)
    x.check(o, state, scale=scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kh,dk,dv,lens", [(2, 1, 128, 128, [1500, 40, 700]), (1, 1, 64, 80, [2100]), (2, 2, 256, 64, [900, 1025])])
def test_growing_decays_in_segments(t, heads, kh, dk, dv, lens):
    """Bursts that grow by e^32 and fall again, so that segments begin and end anywhere in them."""
    x = Linear(_gen(dk), t, heads, kh, dk, dv, lens)
    wave = torch.where(torch.arange(x.g.shape[0], device="cuda") % 128 < 64, 0.5, -0.55)
    x.g = wave[:, None].expand(-1, heads).contiguous()
    scale = _scale(x)
    o, state, need = x.run(scale=scale)
    assert need > 0
    x.check(o, state, scale=scale)


@pytest.mark.parametrize("t", TYPES)
def test_decays_of_segments_past_fp32(t):
    """The decay of a segment is below 2^-149, or above 2^128; a state of 2^120 and one of zeros."""
    x = Linear(_gen(67), t, 1, 1, 64, 80, [2100, 300])
    x.v[:] = 0
    x.g[:] = 0
    x.g[256:512], x.g[600:856] = -0.41, 0.38
    x.state[0] *= 2.0 ** 120
    o, state, need = x.run(scale=2.0 ** -122)
    assert need > 0 and float(state[x.to[0]].abs().max()) > 0
    x.check(o, state, scale=2.0 ** -122)
    x.g[:] = 0.38
    x.state[:] = 0
    o, state, _ = x.run()
    assert (o[:2400] == 0).all() and (state == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("lens", [[90, 5], [70, 130]])
def test_values_far_from_states(t, max_new, lens):
    """States near fp32's largest number and values near fp16's smallest: neither is scaled out of its range, and where a
    value meets a state of nothing beside a huge one it keeps its precision."""
    for size, value in ((2.0 ** 92, 2.0 ** -22), (2.0 ** 110, 2.0 ** -14), (2.0 ** 100, 1.0)):
        x = Linear(_gen(61), t, 2, 2, 64, 64, lens)
        x.v, x.state = (x.v.float() * value).to(x.dt), x.state * size
        x.state[:, :, 5:9] = 0
        x.g = 0.01 * x.g
        scale = _scale(x)
        o, state, _ = x.run(scale=scale, max_new=max_new)
        x.check(o, state, scale=scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
def test_states_that_rise_and_fall(t, max_new):
    """A chunk that grows by e^60, then ones that shrink by as much, values of nothing and small ones behind."""
    x = Linear(_gen(62), t, 2, 1, 64, 48, [320])
    x.g = torch.zeros_like(x.g)
    x.g[:60], x.g[64:128], x.g[200:260] = 1.0, -1.0, 0.9
    x.v[64:200] = 0
    x.v[200:] *= 2.0 ** -10
    scale = _scale(x)
    o, state, _ = x.run(scale=scale, max_new=max_new)
    x.check(o, state, scale=scale)


@pytest.mark.parametrize("max_new", [0, 1])
def test_scores_past_every_16_bit_number(max_new):
    """fp16 queries and keys of hundreds over decays of e^70: a channel of zeros stays zero, the others hold."""
    x = Linear(_gen(63), "f16", 1, 1, 64, 64, [70, 20])
    x.q, x.k = x.q * 200, x.k * 100
    x.v[:, :, 7:20] = 0
    x.state[:, :, :, 7:20] = 0
    x.g = torch.full_like(x.g, 1.0)
    scale = _scale(x)
    o, state, _ = x.run(scale=scale, max_new=max_new)
    assert (o[:90, :, 7:20] == 0).all()
    x.check(o, state, scale=scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
def test_what_is_forgotten_does_not_grow_again(t, max_new):
    """A decay of 0, then decays above 1: what was before stays gone."""
    x = Linear(_gen(64), t, 1, 1, 64, 64, [90])
    x.state = x.state * 1e30
    x.v[:] = 0
    x.g[:], x.g[3] = 0.0, -math.inf
    x.g[4:64] = 1.3
    o, state, _ = x.run(scale=1.0, max_new=max_new)
    assert (o[3:90] == 0).all() and (state[x.to[0]] == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("which", ["k", "v", "kv", "q", "near"])
def test_rows_on_top_of_one_another(t, max_new, which):
    """Keys, values and queries broadcast over tokens (a stride of 0), or rows that begin 16 bytes behind one another."""
    x = Linear(_gen(65), t, 2, 2, 64, 64, [70, 1, 64, 9])
    n = x.q.shape[0]
    for name in "qkv" if which == "near" else which:
        rows = getattr(x, name)
        setattr(x, name, rows.flatten().as_strided((n, 2, 64), (8, 64, 1)) if which == "near" else rows[:1].expand(n, -1, -1))
    o, state, _ = x.run(max_new=max_new)
    x.check(o, state)


def test_the_same_call_gives_the_same_bits():
    """Chunks, segments and single tokens, again and again."""
    for t in TYPES:
        for heads, kh, dk, dv, lens, max_new in ((4, 2, 128, 128, [65, 0, 1, 63, 2], 0), (2, 1, 128, 96, [1500, 40, 700], 0), (3, 3, 48, 80, [130, 17], 1),
                                                 (2, 2, 256, 64, [900, 1025], 0)):
            x = Linear(_gen(66), t, heads, kh, dk, dv, lens)
            first = x.run(max_new=max_new)
            for _ in range(5):
                again = x.run(max_new=max_new)
                assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
