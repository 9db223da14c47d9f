"""Attention with shared first tokens, linear attention and sampling: arguments that are refused, on the host before
anything is enqueued, what an empty call does, and workspaces.  No device is needed: every check here comes before the
first HIP call."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

import infvino_amd as ia
from infvino_amd import ops

A = 4096  # stands for device addresses: multiples of 16


def _cache(**kw):
    return ops.cache_desc(**{"type": ops.F16, "bits": 8, "heads": 2, "dim": 64, "page": 16, "pages": 10, "table_width": 8, **kw})


def _prefix(d, args=None, batch=2, groups=1, tokens=2, ws=A, ws_bytes=1 << 40):
    ops.prefix_attention(d, *(args or [A] * 11), batch, groups, tokens, ws, ws_bytes)


@pytest.mark.parametrize("kw,msg", [({"heads": 3}, "multiple"), ({"heads": 0}, "multiple"), ({"scale": float("nan")}, "finite"), ({"scale": 3e38}, "finite"),
                                    ({"max_new": -1}, "negative"), ({"max_len": -1}, "negative"), ({"max_shared": -1}, "negative"),
                                    ({"q": (129, 64)}, "16 bytes"), ({"o": (64, 64)}, "overlap"), ({"o": (256, 32)}, "overlap")])
def test_prefix_attention_refuses(kw, msg):
    d = ops.prefix_attention_desc(_cache(), **{"heads": 4, "scale": 0.1, **kw})
    with pytest.raises(RuntimeError, match=msg):
        _prefix(d)


@pytest.mark.parametrize("kw,msg", [({"type": 2}, "type"), ({"bits": 4}, "bits"), ({"heads": 0}, "heads"), ({"dim": 72}, "dim"), ({"page": 24}, "page"),
                                    ({"pages": 0}, "pages"), ({"table_width": 1 << 27}, "2\\^30")])
def test_prefix_attention_refuses_caches(kw, msg):
    c = _cache(**kw)
    with pytest.raises(RuntimeError, match=msg):
        ops.prefix_attention_workspace(ops.prefix_attention_desc(c, max(c.heads, 1), 1.0), 1, 1, 1)


def test_prefix_attention_refuses_operands_and_workspace():
    d = ops.prefix_attention_desc(_cache(), 4, 0.1)
    need = ops.prefix_attention_workspace(d, 2, 1, 2)
    assert need > 0
    for at in range(11):
        args = [A] * 11
        args[at] = None
        with pytest.raises(RuntimeError, match="null|scales"):
            _prefix(d, args)
    for at, by in ((0, 8), (1, 8), (2, 4), (3, 2), (5, 2), (6, 1), (7, 2), (8, 2), (9, 2), (10, 8)):
        args = [A] * 11
        args[at] = A + by
        with pytest.raises(RuntimeError, match="16 bytes|misaligned"):
            _prefix(d, args)
    for ws, n in ((None, need), (A, need - 1), (A, 0)):
        with pytest.raises(RuntimeError, match="workspace too small"):
            _prefix(d, ws=ws, ws_bytes=n)
    with pytest.raises(RuntimeError, match="workspace must start"):
        _prefix(d, ws=A + 8, ws_bytes=need)
    for batch, groups, tokens, msg in ((-1, 1, 1, "batch"), (1, -1, 1, "groups"), (1, (1 << 20) + 1, 1, "groups"), (1, 1, -1, "tokens"), (1, 1, 1 << 25, "too many rows")):
        with pytest.raises(RuntimeError, match=msg):
            ops.prefix_attention_workspace(d, batch, groups, tokens)
    with pytest.raises(RuntimeError, match="too many rows"):
        ops.prefix_attention_workspace(ops.prefix_attention_desc(_cache(heads=64), 64, 0.1), 1, 1 << 17, 1)
    with pytest.raises(RuntimeError, match="null descriptor"):
        ia._check(ia.lib().ivh_prefix_attention_workspace(None, 1, 1, 1, C.byref(C.c_size_t())))
    with pytest.raises(RuntimeError, match="null bytes"):
        ia._check(ia.lib().ivh_prefix_attention_workspace(d, 1, 1, 1, None))


def test_prefix_attention_splits_fit_a_launch():
    """Work-groups of every kind of call: fewer than 2^24 of 256 lanes, rows of the largest calls among them."""
    for heads, kv, batch, groups, tokens in ((64, 1, 1 << 20, 1 << 20, 1 << 20), (1, 1, 1 << 20, 1, 1 << 26), (4096, 4096, 1 << 10, 1 << 10, 1 << 14), (32, 8, 1, 1, 1 << 21)):
        for width in (8, 1 << 20):
            d = ops.prefix_attention_desc(_cache(heads=kv, table_width=width), heads, 0.1, max_new=1)
            need = ops.prefix_attention_workspace(d, batch, groups, tokens)
            assert need % (tokens * heads * 66 * 4) == 0
            assert 1 <= need // (tokens * heads * 66 * 4) <= 512


def _linear(d, args=None, batch=2, tokens=4, ws=A, ws_bytes=1 << 40):
    ops.linear_attention(d, *(args or [A] * 9), batch, tokens, ws, ws_bytes)


def _linear_desc(**kw):
    return ops.linear_attention_desc(**{"type": ops.BF16, "heads": 4, "key_heads": 2, "key_dim": 64, "dim": 32, "scale": 0.1, "slots": 4, **kw})


@pytest.mark.parametrize("kw,msg", [({"type": 2}, "type"), ({"heads": 3}, "multiple"), ({"key_heads": 0}, "multiple"), ({"heads": 8192, "key_heads": 1}, "multiple"),
                                    ({"key_dim": 24}, "multiples of 16"), ({"key_dim": 272}, "256"), ({"dim": 0}, "multiples of 16"), ({"dim": 8}, "multiples of 16"),
                                    ({"scale": float("inf")}, "finite"), ({"slots": -1}, "slots"), ({"max_new": -1}, "max_new"), ({"g": (-1, 1)}, "decays"),
                                    ({"q": (130, 64)}, "16 bytes"), ({"k": (128, 60)}, "16 bytes"), ({"v": (-128, 32)}, "16 bytes"), ({"o": (64, 32)}, "overlap"),
                                    ({"q": (1 << 23, 64)}, "2\\^23"), ({"v": (1 << 24, 32)}, "2\\^23")])
def test_linear_attention_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        _linear(_linear_desc(**kw))


def test_linear_attention_refuses_operands_and_workspace():
    d = _linear_desc()
    for at in (0, 1, 2, 3, 4, 7, 8):
        args = [A] * 9
        args[at] = None
        with pytest.raises(RuntimeError, match="null"):
            _linear(d, args)
    for at, by in ((0, 8), (1, 8), (2, 8), (3, 2), (4, 2), (5, 1), (6, 2), (7, 8), (8, 8)):
        args = [A] * 9
        args[at] = A + by
        with pytest.raises(RuntimeError, match="16 bytes|misaligned"):
            _linear(d, args)
    long = _linear_desc()
    need = ops.linear_attention_workspace(long, 1, 20000)
    assert need > 0
    for ws, n in ((None, need), (A, need - 1)):
        with pytest.raises(RuntimeError, match="workspace too small"):
            _linear(long, batch=1, tokens=20000, ws=ws, ws_bytes=n)
    with pytest.raises(RuntimeError, match="workspace must start"):
        _linear(long, batch=1, tokens=20000, ws=A + 8, ws_bytes=need)
    for batch, tokens, msg in ((-1, 1, "batch"), (1, -1, "tokens"), (1 << 21, 1, "batch"), (1 << 20, 1, "too many states"), (1 << 18, 1, None)):
        if msg:
            with pytest.raises(RuntimeError, match=msg):
                ops.linear_attention_workspace(d, batch, tokens)
        else:
            ops.linear_attention_workspace(d, batch, tokens)
    with pytest.raises(RuntimeError, match="too many states"):
        ops.linear_attention_workspace(_linear_desc(heads=64, key_heads=64), 1 << 17, 1)
    with pytest.raises(RuntimeError, match="null descriptor"):
        ia._check(ia.lib().ivh_linear_attention_workspace(None, 1, 1, C.byref(C.c_size_t())))


def test_linear_attention_workspace_follows_the_split():
    """One long sequence is cut into segments, short or many ones are not."""
    d = _linear_desc(max_new=1)
    assert ops.linear_attention_workspace(d, 1, 1 << 20) == 0
    assert ops.linear_attention_workspace(_linear_desc(max_new=200), 7, 1400) == 0
    assert ops.linear_attention_workspace(_linear_desc(max_new=2048), 512, 512 * 2048) == 0
    assert ops.linear_attention_workspace(_linear_desc(max_new=16384), 1, 16384) > 0
    for batch, tokens in ((1, 1 << 26), (1 << 18, 1 << 26), (1, 17), (3, 1 << 20)):
        need = ops.linear_attention_workspace(_linear_desc(), batch, tokens)
        assert need % 4 == 0


def _sample(d, args=None, rows=3, ws=A, ws_bytes=1 << 40):
    ops.sample(d, *(args or [A] * 7), rows, ws, ws_bytes)


@pytest.mark.parametrize("kw,msg", [({"type": 3}, "type"), ({"type": -1}, "type"), ({"vocab": 0}, "vocab"), ({"vocab": (1 << 19) + 1}, "vocab"), ({"row": -1}, "stride")])
def test_sample_refuses(kw, msg):
    d = ops.sample_desc(**{"type": ops.F32, "vocab": 100, **kw})
    with pytest.raises(RuntimeError, match=msg):
        _sample(d)
    with pytest.raises(RuntimeError, match=msg):
        ops.sample_workspace(d, 1)


def test_sample_refuses_operands_and_workspace():
    d = ops.sample_desc(ops.F32, 20000)
    for at in (0, 5, 6):
        args = [A] * 7
        args[at] = None
        with pytest.raises(RuntimeError, match="null"):
            _sample(d, args)
    for at in range(7):
        args = [A] * 7
        args[at] = A + 2
        with pytest.raises(RuntimeError, match="misaligned"):
            _sample(d, args)
    with pytest.raises(RuntimeError, match="misaligned"):
        _sample(ops.sample_desc(ops.F16, 20000), [A + 1] + [A] * 6)
    need = ops.sample_workspace(d, 3)
    assert need > 0 and ops.sample_workspace(ops.sample_desc(ops.F32, 8192), 3) == 0
    for ws, n in ((None, need), (A, need - 1)):
        with pytest.raises(RuntimeError, match="workspace too small"):
            _sample(d, ws=ws, ws_bytes=n)
    with pytest.raises(RuntimeError, match="workspace must start"):
        _sample(d, ws=A + 4, ws_bytes=need)
    for rows in (-1, (1 << 20) + 1):
        with pytest.raises(RuntimeError, match="rows"):
            ops.sample_workspace(d, rows)
    with pytest.raises(RuntimeError, match="null descriptor"):
        ia._check(ia.lib().ivh_sample_workspace(None, 1, C.byref(C.c_size_t())))


def test_empty_calls_do_nothing():
    d = ops.prefix_attention_desc(_cache(), 4, 0.1)
    assert ops.prefix_attention_workspace(d, 0, 0, 0) == 0
    _prefix(d, [None] * 11, 0, 0, 0, None, 0)
    _prefix(d, [None] * 11, 3, 1, 0, None, 0)
    _linear(_linear_desc(), [None] * 9, 0, 0, None, 0)
    _sample(ops.sample_desc(ops.F32, 20000), [None] * 7, 0, None, 0)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_structs_have_the_layout_of_the_header(tmp_path):
    """Size of each descriptor, and place and size of each of its fields, as a C compiler has them from include/ivh.h."""
    mirrors = {"ivh_prefix_attn_desc": ia.PrefixAttentionDesc, "ivh_linear_attn_desc": ia.LinearAttentionDesc, "ivh_sample_desc": ia.SampleDesc}
    lines, want = [], []
    for name, mirror in mirrors.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append([C.sizeof(mirror)])
        for field, *_ in mirror._fields_:
            at = getattr(mirror, field)
            lines.append(f'printf("%zu %zu\\n", offsetof({name}, {field}), sizeof(({name} *)0)->{field});'.replace(f"sizeof(({name} *)0)->{field}", f"sizeof((({name} *)0)->{field})"))
            want.append([at.offset, at.size])
    source = tmp_path / "layout.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include <ivh.h>\nint main(void)\n{\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-I", include, str(source), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert [[int(x) for x in line.split()] for line in out.splitlines()] == want
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(include, "ivh.h")).read(), flags=re.S)
    for name, mirror in mirrors.items():
        body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
        fields = [re.search(r"(\w+)(\[\d+\])?$", x.strip()).group(1) for line in body.split("{")[1].split(";")[:-1] for x in line.split(",")]
        assert fields == [x[0] for x in mirror._fields_]
