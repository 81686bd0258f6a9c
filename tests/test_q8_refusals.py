"""What the operators of a decoder layer in 8 bits refuse, before they touch a device, and their structs' layout."""
import ctypes as C
import os
import subprocess

import pytest

from common_b200 import native

ARG, SHAPE, UNSUPPORTED = 1, 2, 8
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def refused(status, call, **over):
    with pytest.raises(native.QwenError) as e:
        call(**over)
    assert e.value.status == status and str(e.value)


def norm(**over):
    n = native.NormQ8(64, 16)
    call = dict(x=16, q=16, scale=16, rows=1)
    for k, v in over.items():
        if k in ("dim", "norm_w", "eps", "x_dtype", "delta_dtype"):
            setattr(n.args, k, v)
        else:
            call[k] = v
    n(**call)


@pytest.mark.parametrize("status,over", [
    (ARG, dict(x=0)), (ARG, dict(norm_w=0)), (ARG, dict(q=0)), (ARG, dict(scale=0)), (ARG, dict(x=18)),
    (ARG, dict(sum_out=18)), (ARG, dict(delta=17)), (ARG, dict(norm_w=18)), (ARG, dict(scale=18)), (ARG, dict(eps=-1.0)),
    (ARG, dict(eps=float("nan"))), (ARG, dict(delta=17, delta_dtype=native.DTYPE_BF16)),
    (ARG, dict(sum_out=16, ld_sum=128)), (ARG, dict(delta=32, sum_out=32, ld_delta=72)),
    (ARG, dict(delta=32, sum_out=32, delta_dtype=native.DTYPE_BF16)),
    (UNSUPPORTED, dict(x_dtype=native.DTYPE_F64)), (UNSUPPORTED, dict(delta=16, delta_dtype=native.DTYPE_F64)),
    (SHAPE, dict(rows=-1)), (SHAPE, dict(dim=0)), (SHAPE, dict(ld_x=63)), (SHAPE, dict(delta=16, ld_delta=63)),
    (SHAPE, dict(sum_out=16, ld_sum=63)), (SHAPE, dict(ld_q=63)), (SHAPE, dict(ld_q=-64)), (SHAPE, dict(dim=(1 << 30) + 1)),
])
def test_norm_refuses(status, over):
    refused(status, norm, **over)


def quant(**over):
    a = dict(x_ptr=16, x_dtype=native.DTYPE_BF16, rows=1, dim=64, q_ptr=16, scale_ptr=16)
    a.update(over)
    native.op_quant_q8(**a)


@pytest.mark.parametrize("status,over", [
    (ARG, dict(x_ptr=0)), (ARG, dict(q_ptr=0)), (ARG, dict(scale_ptr=0)), (ARG, dict(x_ptr=17)), (ARG, dict(scale_ptr=18)),
    (UNSUPPORTED, dict(x_dtype=native.DTYPE_F64)), (SHAPE, dict(rows=-1)), (SHAPE, dict(dim=0)), (SHAPE, dict(ld_x=63)),
    (SHAPE, dict(ld_q=63)),
])
def test_quant_refuses(status, over):
    refused(status, quant, **over)


def linear(**over):
    a = native.LinearQ8(16, 16, 64, 64)
    call = dict(x=16, x_scale=16, t=1, out=16)
    for k, v in over.items():
        if k in ("w", "w_scale", "n_out", "k", "ld_w", "epi", "bias", "out_dtype"):
            setattr(a.args, k, v)
        else:
            call[k] = v
    a(**call)


@pytest.mark.parametrize("status,over", [
    (ARG, dict(w=0)), (ARG, dict(w_scale=0)), (ARG, dict(x=0)), (ARG, dict(x_scale=0)), (ARG, dict(out=0)),
    (ARG, dict(w=8)), (ARG, dict(x=24)), (ARG, dict(out=18)), (ARG, dict(w_scale=18)), (ARG, dict(x_scale=17)),
    (ARG, dict(bias=18)), (ARG, dict(err=18)), (ARG, dict(out=17, out_dtype=native.DTYPE_BF16)),
    (ARG, dict(epi=3)), (ARG, dict(epi=-1)), (ARG, dict(epi=native.LINEAR_RESID)),
    (ARG, dict(epi=native.LINEAR_RESID, resid=18)), (ARG, dict(epi=native.LINEAR_RESID, resid=16, bias=16)),
    (ARG, dict(epi=native.LINEAR_RESID, resid=16, ld_resid=80)),
    (ARG, dict(epi=native.LINEAR_SWIGLU, out_dtype=native.DTYPE_BF16, bias=16)),
    (UNSUPPORTED, dict(out_dtype=native.DTYPE_F64)), (UNSUPPORTED, dict(epi=native.LINEAR_SWIGLU)),
    (UNSUPPORTED, dict(epi=native.LINEAR_RESID, resid=16, out_dtype=native.DTYPE_BF16)),
    (SHAPE, dict(n_out=0)), (SHAPE, dict(t=-1)), (SHAPE, dict(n_out=(1 << 30) + 1)), (SHAPE, dict(t=(1 << 30) + 1)),
    (SHAPE, dict(n_out=1 << 28, t=1 << 12)), (SHAPE, dict(k=0)), (SHAPE, dict(k=131072, ld_w=131072, ld_x=131072)),
    (SHAPE, dict(k=60)), (SHAPE, dict(ld_w=48)), (SHAPE, dict(ld_w=72)), (SHAPE, dict(ld_x=72)), (SHAPE, dict(ld_x=1 << 31)),
    (SHAPE, dict(ld_out=63)), (SHAPE, dict(epi=native.LINEAR_RESID, resid=16, ld_resid=63)),
    (SHAPE, dict(epi=native.LINEAR_SWIGLU, out_dtype=native.DTYPE_BF16, n_out=48)),
])
def test_linear_refuses(status, over):
    refused(status, linear, **over)


def append(**over):
    a = native.KvAppend(16, 8, 128, 64, 10, 4, rope=16, rope_len=8)
    call = dict(q=16, k=16, v=16, q_out=32, k_cache=16, v_cache=16, page_table=16, row_start=16, kv_len=16, batch=1, rows=1)
    for k, v in over.items():
        if k in call or k in ("ld_q", "ld_k", "ld_v", "ld_q_out"):
            call[k] = v
        else:
            setattr(a.args, k, v)
    a(**call)


@pytest.mark.parametrize("status,over", [
    (ARG, dict(q=0)), (ARG, dict(k=0)), (ARG, dict(v=0)), (ARG, dict(k_cache=0)), (ARG, dict(v_cache=0)),
    (ARG, dict(page_table=0)), (ARG, dict(row_start=0)), (ARG, dict(kv_len=0)), (ARG, dict(q=8)), (ARG, dict(k=24)),
    (ARG, dict(q_out=8)), (ARG, dict(k_cache=8)), (ARG, dict(rope=8)), (ARG, dict(qk_norm=3)),
    (ARG, dict(qk_norm=native.QKNORM_HEAD)), (ARG, dict(qk_norm=native.QKNORM_HEAD, q_norm=16)),
    (ARG, dict(qk_norm=native.QKNORM_HEAD, q_norm=16, k_norm=8)), (ARG, dict(eps=-1e-6)), (ARG, dict(q_out=16)),
    (ARG, dict(q_out=16, in_dtype=native.DTYPE_BF16, ld_q=4096)),
    (UNSUPPORTED, dict(in_dtype=native.DTYPE_F64)), (UNSUPPORTED, dict(dtype=native.DTYPE_F64)),
    (UNSUPPORTED, dict(head_dim=96)), (UNSUPPORTED, dict(head_dim=512)), (UNSUPPORTED, dict(head_dim=8)),
    (SHAPE, dict(heads=0)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(heads=497)), (SHAPE, dict(batch=-1)),
    (SHAPE, dict(batch=1025)), (SHAPE, dict(rows=-1)), (SHAPE, dict(page_size=48)), (SHAPE, dict(page_size=512)),
    (SHAPE, dict(num_pages=0)), (SHAPE, dict(max_pages=0)), (SHAPE, dict(max_pages=1 << 25)), (SHAPE, dict(rope_len=0)),
    (SHAPE, dict(ld_q=2040)), (SHAPE, dict(ld_k=1026)), (SHAPE, dict(ld_v=1000)), (SHAPE, dict(ld_q_out=2052)),
])
def test_append_refuses(status, over):
    refused(status, append, **over)


def test_nothing_is_done():
    norm(rows=0, x=0)
    quant(rows=0, x_ptr=0)
    linear(t=0, x=0)
    append(rows=0, q=0)
    append(batch=0, row_start=0)


def test_null_arguments():
    lib = native.load()
    for fn in (lib.qw_op_norm_q8, lib.qw_op_linear_q8, lib.qw_op_kv_append):
        assert fn(None, None) == ARG


def test_struct_layouts_match_c(tmp_path):
    structs = {"qw_norm_q8_args": native.NormQ8Args, "qw_linear_q8_args": native.LinearQ8Args,
               "qw_kv_append_args": native.KvAppendArgs}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src, exe = tmp_path / "t.c", str(tmp_path / "t")
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"qwen3_b200.h\"\nint main(void) {\n" +
                   "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["/usr/bin/gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = list(map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()))
    want = []
    for cls in structs.values():
        want += [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
