"""What the operators of the paged cache refuse, before they touch a device."""
import pytest

from common_b200 import native

ARG, SHAPE, UNSUPPORTED = 1, 2, 8


def attention(**over):
    a = native.ChunkAttention(16, 8, 128, 64, 10, 4, 256, 1 << 40)
    for k in list(over):
        if k in dict(a.args._fields_) and k not in ("q", "k_cache", "v_cache", "page_table", "row_start", "kv_len",
                                                    "batch", "rows", "out", "lse", "ld_q", "ld_out"):
            setattr(a.args, k, over.pop(k))
    call = dict(q=16, k_cache=16, v_cache=16, page_table=16, row_start=16, kv_len=16, batch=1, rows=1, out=16)
    call.update(over)
    a(**call)


@pytest.mark.parametrize("status,over", [
    (ARG, dict(q=0)), (ARG, dict(k_cache=0)), (ARG, dict(v_cache=0)), (ARG, dict(page_table=0)),
    (ARG, dict(row_start=0)), (ARG, dict(kv_len=0)), (ARG, dict(out=0)), (ARG, dict(workspace=0)),
    (ARG, dict(workspace=264)), (ARG, dict(workspace_bytes=16)), (ARG, dict(q=18)), (ARG, dict(out=24)),
    (ARG, dict(k_cache=8)), (ARG, dict(window=-1)), (ARG, dict(scale=-1.0)), (ARG, dict(scale=float("inf"))),
    (ARG, dict(scale=float("nan"))), (UNSUPPORTED, dict(dtype=native.DTYPE_F64)), (UNSUPPORTED, dict(head_dim=96)),
    (SHAPE, dict(heads=12)), (SHAPE, dict(heads=136)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(batch=-1)),
    (SHAPE, dict(batch=1025)), (SHAPE, dict(rows=-1)), (SHAPE, dict(page_size=8)), (SHAPE, dict(page_size=48)),
    (SHAPE, dict(page_size=512)), (SHAPE, dict(num_pages=0)), (SHAPE, dict(max_pages=0)),
    (SHAPE, dict(max_pages=1 << 25)), (SHAPE, dict(num_pages=1 << 23)), (SHAPE, dict(ld_q=2040)),
    (SHAPE, dict(ld_q=2052)), (SHAPE, dict(ld_out=1024)),
])
def test_chunk_attention_refuses(status, over):
    with pytest.raises(native.QwenError) as e:
        attention(**over)
    assert e.value.status == status and str(e.value)


def test_chunk_attention_refuses_more_key_blocks_than_it_can_number():
    # 2^22 rows over 2^22 positions: 2^16 items of 2^15 blocks, two tiles, 8 KV heads
    with pytest.raises(native.QwenError) as e:
        attention(rows=1 << 22, max_pages=1 << 16)
    assert e.value.status == SHAPE and "key blocks" in str(e.value)


def test_chunk_attention_of_nothing_is_done():
    attention(rows=0, q=0)
    attention(batch=0, row_start=0)


def test_workspace_refuses_unknown_geometries():
    for g in ((16, 8, 96), (12, 8, 128), (16, 0, 128)):
        with pytest.raises(native.QwenError):
            native.chunk_attn_workspace(*g)
    assert native.chunk_attn_workspace(16, 8, 128) >= 256


def test_null_arguments():
    lib = native.load()
    assert lib.qw_op_chunk_attn(None, None) == ARG
    assert lib.qw_op_kv_copy_pages(None, None, None, None, 1, None) == ARG
    assert lib.qw_op_kv_compact(None, None, None, 1, None, None, None, 1, 1, None, 0, None) == ARG


def pool(**over):
    f = dict(k=16, v=16, layers=2, num_pages=4, kv_heads=2, page_size=64, head_dim=128, dtype=native.DTYPE_BF16)
    f.update(over)
    return native.KvPool(*[f[n] for n, _ in native.KvPool._fields_])


@pytest.mark.parametrize("status,over", [
    (ARG, dict(k=0)), (ARG, dict(v=0)), (ARG, dict(k=8)), (UNSUPPORTED, dict(dtype=native.DTYPE_F64)),
    (SHAPE, dict(layers=0)), (SHAPE, dict(num_pages=0)), (SHAPE, dict(kv_heads=0)), (SHAPE, dict(head_dim=40)),
    (SHAPE, dict(page_size=0)), (SHAPE, dict(page_size=96)), (SHAPE, dict(page_size=512)), (SHAPE, dict(layers=40000)),
])
def test_page_operators_refuse_a_pool(status, over):
    with pytest.raises(native.QwenError) as e:
        native.op_kv_copy_pages(pool(**over), 16, 16, 16, 1)
    assert e.value.status == status
    with pytest.raises(native.QwenError) as e:
        native.op_kv_compact(pool(**over), 16, 16, 4, 16, 16, 1, 1)
    assert e.value.status == status


def test_page_operators_refuse_bad_arguments():
    p = pool()
    for status, call in [
        (ARG, lambda: native.op_kv_copy_pages(p, 0, 16, 0, 1)), (ARG, lambda: native.op_kv_copy_pages(p, 16, 0, 0, 1)),
        (SHAPE, lambda: native.op_kv_copy_pages(p, 16, 16, 0, -1)),
        (ARG, lambda: native.op_kv_compact(p, 0, 16, 4, 16, 16, 1, 1)),
        (ARG, lambda: native.op_kv_compact(p, 16, 0, 4, 16, 16, 1, 1)),
        (ARG, lambda: native.op_kv_compact(p, 16, 16, 4, 0, 16, 1, 1)),
        (ARG, lambda: native.op_kv_compact(p, 16, 16, 4, 16, 0, 1, 1)),
        (ARG, lambda: native.op_kv_compact(p, 16, 16, 4, 16, 16, 1, 1, rope=24, rope_len=4)),
        (SHAPE, lambda: native.op_kv_compact(p, 16, 16, 4, 16, 16, 1, 1, rope=16, rope_len=0)),
        (SHAPE, lambda: native.op_kv_compact(p, 16, 16, 4, 16, 16, 0, 1)),
        (SHAPE, lambda: native.op_kv_compact(p, 16, 16, 0, 16, 16, 1, 1)),
        (SHAPE, lambda: native.op_kv_compact(p, 16, 16, 4, 16, 16, 1, -1)),
    ]:
        with pytest.raises(native.QwenError) as e:
            call()
        assert e.value.status == status
    native.op_kv_copy_pages(p, 0, 0, 0, 0)
    native.op_kv_compact(p, 0, 0, 4, 0, 0, 1, 0)
