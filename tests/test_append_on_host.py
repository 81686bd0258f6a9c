"""The append's kernels (qw_kv_append.cu) compiled for the host and run there, in buffers that end where a page without access
begins: a read or write past them ends the process with a signal, without a GPU.  host_cuda/ holds what stands for CUDA."""
import os
import re
import subprocess

import pytest

from common_b200 import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "common_b200", "csrc")
HOST = os.path.join(ROOT, "tests", "host_cuda")
NONE, VECTOR, HEAD = native.QKNORM_NONE, native.QKNORM_VECTOR, native.QKNORM_HEAD
F32, BF16 = native.DTYPE_F32, native.DTYPE_BF16


@pytest.fixture(scope="module")
def append(tmp_path_factory):
    """The kernels' source without its inline assembly, its shared memory from the launch, as a program of the host."""
    tmp = tmp_path_factory.mktemp("host")
    to = tmp / "common_b200" / "csrc"
    to.mkdir(parents=True)
    for name in ("qw_kv_append.cu", "qw_internal.cuh", "qw_ops.h", "qw_chunk_attn.h"):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        text = re.sub(r"\basm( volatile)?\(.*?\);", "", text, flags=re.S)
        text = re.sub(r"extern __shared__ __align__\(16\) (\w+) (\w+)\[\];", r"\1 *\2 = (\1 *)host_dynamic_shared;", text)
        (to / name).write_text(text)
    (tmp / "include").symlink_to(os.path.join(ROOT, "include"))
    exe = str(tmp / "append")
    # without optimisation: every load of the source is made
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O0", "-fno-strict-aliasing", f"-I{HOST}", f"-I{tmp}",
                    os.path.join(HOST, "append.cpp"), "-o", exe], check=True)
    return lambda *args: subprocess.run([exe] + [str(int(a)) for a in args], capture_output=True, text=True, timeout=600)


def check(run):
    assert run.returncode == 0, (run.returncode, run.stderr)


# heads that fill the lanes' groups, and that leave a round of them short
GEOMETRIES = [(16, 8, 128), (32, 8, 128), (28, 4, 128), (12, 2, 128), (14, 2, 64), (8, 1, 64), (12, 8, 128), (3, 1, 16),
              (4, 4, 32), (6, 2, 256), (1, 1, 128), (2, 5, 64)]


@pytest.mark.parametrize("mode", [NONE, HEAD, VECTOR])
@pytest.mark.parametrize("heads,kv_heads,d", GEOMETRIES)
def test_few_rows(append, heads, kv_heads, d, mode):
    check(append(heads, kv_heads, d, 45, mode, F32, BF16, True, heads % 2, 16, False))


# one, two, three and four rows in the last group
@pytest.mark.parametrize("rows", [1025, 1026, 1027, 1028])
@pytest.mark.parametrize("heads,kv_heads,d", GEOMETRIES)
def test_many_rows(append, heads, kv_heads, d, rows):
    check(append(heads, kv_heads, d, rows, HEAD if rows % 2 else NONE, BF16, BF16, True, rows < 1027, 64, False))


@pytest.mark.parametrize("in_type,out_type", [(F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("turned", [False, True])
def test_types(append, in_type, out_type, turned):
    check(append(14, 2, 64, 1031, HEAD, in_type, out_type, turned, True, 16, False))
    check(append(6, 2, 256, 1030, NONE, in_type, out_type, turned, False, 256, False))


@pytest.mark.parametrize("rows", [40, 1026])
@pytest.mark.parametrize("mode", [NONE, HEAD, VECTOR])
def test_queries_in_place(append, rows, mode):
    check(append(14, 2, 64, rows, mode, F32, F32, True, True, 16, True))
