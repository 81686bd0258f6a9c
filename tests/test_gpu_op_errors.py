"""A launch that fails is reported by the call that made it, and by no call after it."""
import ctypes as C

import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu
CUDA = 4


def broken_capture():
    """(stream, end): a stream whose capture cannot go on, so that launches on it fail on the host; end() ends the capture."""
    import torch
    torch.cuda.init()
    torch.zeros(1, device="cuda")
    cu = C.CDLL("libcuda.so.1")
    stream, graph = C.c_void_p(), C.c_void_p()
    assert cu.cuStreamCreate(C.byref(stream), 1) == 0
    assert cu.cuStreamBeginCapture_v2(stream, 2) == 0
    assert cu.cuStreamSynchronize(stream) != 0  # not allowed while it captures

    def end():
        assert cu.cuStreamEndCapture(stream, C.byref(graph)) != 0
        assert cu.cuStreamDestroy_v2(stream) == 0
    return stream.value, end


def fails(call):
    with pytest.raises(native.QwenError) as e:
        call()
    assert e.value.status == CUDA and "launch" in str(e.value)


def test_failed_launches_leave_no_error():
    import torch
    f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    codes = torch.zeros((64, 64), dtype=torch.int8, device="cuda")
    x, w, s = f(64, 64), f(64), f(64)
    cache = torch.zeros((4, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
    table, start, kv = i(0, 1), i(0, 1), i(1)
    pool = native.KvPool(cache.data_ptr(), cache.data_ptr(), 1, 4, 1, 16, 64, native.DTYPE_BF16)
    a, b = i(0), i(1)
    calls = [
        lambda st: native.NormQ8(64, w.data_ptr())(x.data_ptr(), codes.data_ptr(), s.data_ptr(), 64, stream=st),
        lambda st: native.op_quant_q8(x.data_ptr(), native.DTYPE_F32, 64, 64, codes.data_ptr(), s.data_ptr(), stream=st),
        lambda st: native.LinearQ8(codes.data_ptr(), s.data_ptr(), 64, 64)(codes.data_ptr(), s.data_ptr(), 64, x.data_ptr(), stream=st),
        lambda st: native.KvAppend(1, 1, 64, 16, 4, 2)(x.data_ptr(), x.data_ptr(), x.data_ptr(), 0, cache.data_ptr(), cache.data_ptr(),
                                                      table.data_ptr(), start.data_ptr(), kv.data_ptr(), 1, 1, stream=st),
    ]
    for call in calls:
        stream, end = broken_capture()
        fails(lambda: call(stream))
        end()
        # a call that asks the runtime for its launch's error
        native.op_kv_copy_pages(pool, a.data_ptr(), b.data_ptr(), 0, 1)
        call(0)
    torch.cuda.synchronize()
