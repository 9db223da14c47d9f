"""How calls of the sequence operators are split into launches, on the host alone."""
import os
import subprocess

import pytest

import infvino_amd as ia
from infvino_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.mark.skipif(not os.path.exists(CLANG), reason="no clang++")
def test_launches_hold_their_work_groups(tmp_path):
    """tests/cpp/launch_checks.cpp: grids of the largest calls that are accepted (2^26 rows of any head size among them) and of
    random ones, joins and workspaces included."""
    ia.lib()
    lib, exe = os.path.join(ROOT, "infvino_amd"), str(tmp_path / "launch_checks")
    subprocess.run([CLANG, "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I", os.path.join(lib, "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "launch_checks.cpp"), "-o", exe, "-L", lib, "-linfvino_hip", "-Wl,-rpath," + lib], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout[-500:], r.stderr[-4000:])
    assert r.returncode == 0 and "0 failures" in r.stdout


def test_long_sequences_are_cut_where_they_leave_compute_units_idle():
    """Segments cost a second pass over keys and values: none where whole sequences give each CU a work-group (measured on both
    sides beside linear_split)."""
    for batch, tokens, cut in ((8, 4096, False), (8, 2048, False), (6, 4096, False), (12, 4096, False), (4, 4096, True), (1, 4096, True), (1, 768, True), (1, 300, False)):
        d = ops.linear_attention_desc(ops.BF16, 32, 32, 128, 128, 0.1, batch, max_new=tokens)
        assert (ops.linear_attention_workspace(d, batch, batch * tokens) > 0) == cut, (batch, tokens)
