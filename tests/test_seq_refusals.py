"""Sequence operators (rotary positions, paged cache, attention): arguments that are refused, on the host
before anything is enqueued, and what an empty call does.  No device is needed: every check here comes
before the first HIP call."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

import infvino_amd as ia
from infvino_amd import ops

A = 4096  # stands for device addresses: multiples of 16


@pytest.mark.parametrize("kw,msg", [
    ({"type": 2}, "type"), ({"heads": 0}, "heads"), ({"dim": 60, "sections": (16,)}, "dim"), ({"dim": 1032}, "dim"),
    ({"sections": (34,)}, "rot must"), ({"sections": (6,)}, "rot must"), ({"sections": ()}, "rot must"),
    ({"sections": (16, 16, -4, 4)}, "section"), ({"sections": (16, 8), "rot": 64}, "sum"),
    ({"x": None}, "rope input: null"), ({"y": None}, "rope output: null"), ({"pos": None}, "null positions"),
    ({"freq": None}, "null positions"), ({"x": A + 2}, "multiples of 8 bytes"), ({"y": A + 4}, "multiples of 8 bytes"),
    ({"pos": A + 2}, "misaligned"), ({"xs": (256, 66)}, "multiples of 8 bytes"), ({"ys": (128, 64)}, "overlap"),
    ({"ys": (256, 0)}, "overlap"), ({"xs": (-256, 64)}, "multiples of 8 bytes"), ({"pos_axis": -1}, "stride of positions"),
    ({"tokens": -1}, "tokens"), ({"tokens": (1 << 26) + 1}, "tokens"),
])
def test_rope_refuses(kw, msg):
    strides = {k[0]: kw[k] for k in ("xs", "ys") if k in kw}
    rest = {k: v for k, v in kw.items() if k not in ("xs", "ys")}
    d = {"type": ops.BF16, "heads": 4, "dim": 64, "sections": (32,)}
    call = {k: rest.pop(k) for k in ("x", "y", "pos", "freq", "tokens") if k in rest}
    d.update(rest)
    desc = ops.rope_desc(**d, **strides)
    with pytest.raises(RuntimeError, match=msg):
        ops.rope(desc, call.get("x", A), call.get("pos", A), call.get("freq", A), call.get("y", A), call.get("tokens", 4))


def test_rope_sections_of_absent_axes():
    d = ops.rope_desc(ops.F16, 2, 64, (32,))
    d.rotation.section[2] = 4
    with pytest.raises(RuntimeError, match="section"):
        ops.rope(d, A, A, A, A, 1)
    with pytest.raises(RuntimeError, match="axes"):
        ops.rotation((1, 2, 3, 4, 5))
    with pytest.raises(RuntimeError, match="null descriptor"):
        ia._check(ia.lib().ivh_rope(None, A, A, A, A, 1, None))


def _cache(**kw):
    d = {"type": ops.F16, "bits": 8, "heads": 2, "dim": 64, "page": 16, "pages": 10, "table_width": 8, **kw}
    return ops.cache_desc(**d)


BAD_CACHE = [({"type": 3}, "type"), ({"bits": 4}, "bits"), ({"heads": 0}, "heads"), ({"dim": 72}, "dim"), ({"dim": 272}, "dim"),
             ({"page": 24}, "page"), ({"page": 256}, "page"), ({"pages": 0}, "pages"), ({"table_width": 0}, "pages"),
             ({"table_width": 1 << 27}, "2\\^30")]


@pytest.mark.parametrize("kw,msg", BAD_CACHE)
def test_cache_refuses(kw, msg):
    c = _cache(**kw)
    with pytest.raises(RuntimeError, match=msg):
        ops.cache_bytes(c)
    with pytest.raises(RuntimeError, match=msg):
        ops.kv_append(ops.append_desc(c), A, A, None, None, A, A, A, A, A, A, A, 1, 1)
    with pytest.raises(RuntimeError, match=msg):
        ops.paged_attention_workspace(ops.paged_attention_desc(c, max(c.heads, 1), 1.0), 1, 1)


def test_cache_bytes():
    assert ops.cache_bytes(_cache()) == (10 * 2 * 16 * 64, 10 * 2 * 4)
    assert ops.cache_bytes(_cache(bits=16)) == (10 * 2 * 16 * 64 * 2, 0)
    # sizes past 32 bits
    assert ops.cache_bytes(_cache(heads=128, dim=256, page=128, pages=100000))[0] == 128 * 256 * 128 * 100000


@pytest.mark.parametrize("at,msg", [(0, "keys: null"), (1, "values: null"), (4, "null operand"), (5, "null operand"),
                                    (6, "null operand"), (7, "null operand"), (8, "null operand"), (9, "scales"), (10, "scales")])
def test_append_refuses_null(at, msg):
    args = [A] * 11
    args[at] = None
    with pytest.raises(RuntimeError, match=msg):
        ops.kv_append(ops.append_desc(_cache()), *args, 1, 1)


def test_append_refuses():
    with pytest.raises(RuntimeError, match="null positions"):
        ops.kv_append(ops.append_desc(_cache(), (32,)), A, A, None, A, A, A, A, A, A, A, A, 1, 1)
    with pytest.raises(RuntimeError, match="multiples of 8 bytes"):
        ops.kv_append(ops.append_desc(_cache(), k=(130, 64)), A, A, None, None, A, A, A, A, A, A, A, 1, 1)
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        ops.kv_append(ops.append_desc(_cache()), A, A, None, None, A, A, A, A + 8, A, A, A, 1, 1)
    with pytest.raises(RuntimeError, match="batch"):
        ops.kv_append(ops.append_desc(_cache()), *[A] * 11, -1, 1)
    with pytest.raises(RuntimeError, match="tokens"):
        ops.kv_append(ops.append_desc(_cache()), *[A] * 11, 1, -1)


def _paged(d, args=None, batch=2, tokens=2, ws=None, ws_bytes=0):
    ops.paged_attention(d, *(args or [A] * 9), batch, tokens, ws, ws_bytes)


@pytest.mark.parametrize("kw,msg", [({"heads": 3}, "multiple"), ({"heads": 0}, "multiple"), ({"scale": float("nan")}, "finite"),
                                    ({"scale": float("inf")}, "finite"), ({"window": -1}, "negative"), ({"sinks": -2}, "negative"),
                                    ({"max_new": -1}, "negative"), ({"max_len": -1}, "negative"), ({"q": (129, 64)}, "16 bytes"),
                                    ({"o": (64, 64)}, "overlap"), ({"o": (256, 32)}, "overlap")])
def test_paged_attention_refuses(kw, msg):
    d = ops.paged_attention_desc(_cache(), **{"heads": 4, "scale": 0.1, "max_new": 1, "max_len": 16, **kw})
    with pytest.raises(RuntimeError, match=msg):
        _paged(d)


def test_paged_attention_refuses_operands_and_workspace():
    one = ops.paged_attention_desc(_cache(), 4, 0.1, max_new=1, max_len=16)
    for at in range(9):
        args = [A] * 9
        args[at] = None
        with pytest.raises(RuntimeError, match="null|scales"):
            _paged(one, args)
    many = ops.paged_attention_desc(_cache(table_width=4096, pages=5000), 4, 0.1, max_new=1)
    need = ops.paged_attention_workspace(many, 2, 2)
    assert need > 0
    for ws, n in ((None, need), (A, need - 1), (A, 0)):
        with pytest.raises(RuntimeError, match="workspace"):
            _paged(many, ws=ws, ws_bytes=n)
    with pytest.raises(RuntimeError, match="workspace must start"):
        _paged(many, ws=A + 8, ws_bytes=need)
    with pytest.raises(RuntimeError, match="too many rows"):
        _paged(one, tokens=1 << 25)
    with pytest.raises(RuntimeError, match="too many rows"):
        ops.paged_attention_workspace(ops.paged_attention_desc(_cache(heads=64), 64, 0.1), 1 << 17, 1)
    with pytest.raises(RuntimeError, match="too many rows"):
        ops.attention(ops.attention_desc(ops.F16, 64, 2, 64, 0.1), *[A] * 6, 1 << 17, 4, 4)
    with pytest.raises(RuntimeError, match="finite"):
        ops.paged_attention_workspace(ops.paged_attention_desc(_cache(), 4, 3e38), 1, 1)


@pytest.mark.parametrize("kw,msg", [({"type": -1}, "type"), ({"kv_heads": 3}, "multiple"), ({"kv_heads": 0}, "multiple"),
                                    ({"dim": 264}, "dim"), ({"dim": 12}, "dim"), ({"scale": float("inf")}, "finite"),
                                    ({"window": -1}, "negative"), ({"max_q": -1}, "negative"), ({"k": (1 << 23, 64)}, "2\\^23"),
                                    ({"v": (132, 64)}, "16 bytes"), ({"o": (0, 64)}, "overlap")])
def test_attention_refuses(kw, msg):
    d = ops.attention_desc(**{"type": ops.F16, "heads": 4, "kv_heads": 2, "dim": 64, "scale": 0.1, **kw})
    with pytest.raises(RuntimeError, match=msg):
        ops.attention(d, A, A, A, A, A, A, 1, 4, 4)


def test_attention_refuses_null():
    d = ops.attention_desc(ops.F16, 4, 2, 64, 0.1)
    for at in range(6):
        args = [A] * 6
        args[at] = None
        with pytest.raises(RuntimeError, match="null"):
            ops.attention(d, *args, 1, 4, 4)


def test_empty_calls_do_nothing():
    ops.rope(ops.rope_desc(ops.F16, 2, 64, (32,)), None, None, None, None, 0)
    ops.kv_append(ops.append_desc(_cache()), *[None] * 11, 1, 0)
    ops.kv_append(ops.append_desc(_cache()), *[None] * 11, 0, 3)
    _paged(ops.paged_attention_desc(_cache(), 2, 1.0), [None] * 9, 2, 0)
    ops.attention(ops.attention_desc(ops.F16, 2, 2, 64, 1.0), *[None] * 6, 0, 0, 0)


def test_structs_match_the_header():
    """ctypes mirrors of the descriptors have the sizes a C compiler gives them."""
    assert C.sizeof(ia.Rotation) == 32 and C.sizeof(ia.CacheDesc) == 28
    assert C.sizeof(ia.RopeDesc) == 88 and C.sizeof(ia.AppendDesc) == 104
    assert C.sizeof(ia.PagedAttentionDesc) == 88 and C.sizeof(ia.AttentionDesc) == 104


def test_workspace_follows_the_split():
    """Few rows against many keys are split; many sequences and short ones are not."""
    c = _cache(table_width=4096, pages=5000)
    assert ops.paged_attention_workspace(ops.paged_attention_desc(c, 4, 0.1, max_new=1, max_len=200), 1, 1) == 0
    assert ops.paged_attention_workspace(ops.paged_attention_desc(c, 4, 0.1, max_new=1, max_len=60000), 1, 1) > 0
    assert ops.paged_attention_workspace(ops.paged_attention_desc(c, 4, 0.1, max_new=1, max_len=2000), 2000, 2000) == 0
    # a window bounds what a row reads
    assert ops.paged_attention_workspace(ops.paged_attention_desc(c, 4, 0.1, window=64, max_new=1, max_len=60000), 1, 1) == 0


def test_workspace_of_more_rows_than_a_join_holds():
    """The join of partial sums has a work-group for each row at most, of which a launch holds fewer than
    2^24: calls of more rows are not split."""
    def need(rows, heads, dim):
        c = _cache(heads=1, dim=dim, page=128, table_width=512, pages=1)
        d = ops.paged_attention_desc(c, heads, 0.1, max_new=1, max_len=60000)
        return ops.paged_attention_workspace(d, 1 << 10, rows // heads)

    for dim in (16, 176, 256):
        for heads in (1, 8):
            assert need((1 << 24) - 8, heads, dim) > 0
            assert need(1 << 24, heads, dim) == 0
            assert need(1 << 26, heads, dim) == 0


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_structs_have_the_layout_of_the_header(tmp_path):
    """Size of each descriptor, and place and size of each of its fields, as a C compiler has them from
    include/ivh.h."""
    mirrors = {"ivh_conv_desc": ia.ConvDesc, "ivh_rotation": ia.Rotation, "ivh_rope_desc": ia.RopeDesc, "ivh_cache_desc": ia.CacheDesc,
               "ivh_append_desc": ia.AppendDesc, "ivh_paged_attn_desc": ia.PagedAttentionDesc, "ivh_attn_desc": ia.AttentionDesc}
    lines, want = [], []
    for name, mirror in mirrors.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append([C.sizeof(mirror)])
        for field in mirror._fields_:
            at, kind = getattr(mirror, field[0]), field[1]
            # a float or an integer: halves of 1 differ in whether anything is left
            lines.append(f'{{ {name} d; printf("%zu %zu", offsetof({name}, {field[0]}), sizeof d.{field[0]});')
            want.append([at.offset, at.size])
            if kind in (C.c_int, C.c_int64, C.c_float):
                lines.append(f'd.{field[0]} = 1; d.{field[0]} /= 2; printf(" %d", d.{field[0]} != 0);')
                want[-1].append(int(kind is C.c_float))
            lines.append('printf("\\n"); }')
    source = tmp_path / "layout.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include <ivh.h>\nint main(void)\n{\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-I", include, str(source), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = [[int(x) for x in line.split()] for line in out.splitlines()]
    assert got == want
    # and no field that is not in the mirror
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(include, "ivh.h")).read(), flags=re.S)
    for name, mirror in mirrors.items():
        body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
        fields = [re.search(r"(\w+)(\[\d+\])?$", x.strip()).group(1) for line in body.split("{")[1].split(";")[:-1] for x in line.split(",")]
        assert fields == [x[0] for x in mirror._fields_]
