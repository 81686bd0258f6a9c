"""The chunk attention's workspace after a wait gave up: zeroed again, it serves calls as a new one does, and a model whose
error word is set says so from qw_extend instead of going on.

No wait of the attention kernel is made to run out here.  Its part is played by the counts that such a call can leave, and,
on the model, by the step kernel's test hook (qw_config.test_stall_cta), which sets the same error word."""
import numpy as np
import pytest

from common_b200 import native
from tests.helpers import cfg_dict, rel_l2, state_dict
from tests.test_gpu_chunk_attn import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_workspace_zeroed_again_is_a_new_one(dtype):
    import torch
    c = Case([1, 60], [9001, 2900], 16, 4, 128, 64, dtype=dtype, seed=51)
    c.run()
    c.check()
    out, lse = c.obuf.clone(), c.lse.clone()
    counts = c.ws[: 3 * 256 * 4].view(torch.int32)
    assert not bool(counts.any())                 # a call that ends as it should leaves none
    counts.copy_(torch.arange(768, dtype=torch.int32) % 17)
    c.ws.zero_()
    c.obuf.fill_(-7.0)
    c.run()
    c.check()
    assert torch.equal(out, c.obuf) and torch.equal(lse, c.lse)


def test_extend_reports_a_wait_that_gave_up():
    c = cfg_dict(seq_len=96, dim=512, hidden_dim=1024, heads=8, kv_heads=4, head_dim=64)
    sd = state_dict(c, seed=50, std=0.05)

    def model(**kw):
        m = native.NativeModel(native.make_config(c["dim"], c["hidden_dim"], c["layers"], c["heads"], c["kv_heads"],
                                                  c["head_dim"], c["vocab"], c["seq_len"], False, native.QKNORM_VECTOR, False,
                                                  native.DTYPE_BF16, native.DTYPE_BF16, 1, 64, **kw))
        for k, v in sd.items():
            m.load_tensor(k, v)
        m.finalize()
        return m

    toks = np.arange(40, dtype=np.int32)
    m = model(wait_limit_us=20000, test_stall_cta=6)
    want, _ = m.extend([toks], [0])               # the step kernel has no part in it
    m.decode_step([3], [40], want_logits=False)
    for _ in range(2):
        with pytest.raises(native.QwenError) as e:
            m.extend([toks], [40])
        assert e.value.status == 6
    m.close()
    m = model()
    got, _ = m.extend([toks], [0])
    assert rel_l2(got[0], want[0]) < 2e-2
    m.synchronize()
    m.close()
