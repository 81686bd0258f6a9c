"""The largest numbers of rows that the 8-bit layer's row operators and the append accept: 2^31 - 1, in tens of gigabytes."""
import pytest

from common_b200 import native

pytestmark = pytest.mark.gpu
ROWS = (1 << 31) - 1
AT = [0, 1, 5, 1 << 20, (1 << 30) + 3, ROWS - 5, ROWS - 4, ROWS - 3, ROWS - 2, ROWS - 1]


@pytest.fixture(autouse=True)
def _room():
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("norm", [False, True])
def test_codes(norm):
    """Rows of one bf16 number each, 16 bytes apart: one piece of a lane, four rows a CTA."""
    import torch
    x = torch.zeros((ROWS, 8), dtype=torch.bfloat16, device="cuda")
    q = torch.full((ROWS, 8), 3, dtype=torch.int8, device="cuda")
    scale = torch.full((ROWS,), 7.0, device="cuda")
    for i, r in enumerate(AT):
        x[r, 0] = (-1) ** i * 127.0 * (i + 1)
    if norm:
        w = torch.ones(1, device="cuda")
        native.NormQ8(1, w.data_ptr(), 0.0, native.DTYPE_BF16)(x.data_ptr(), q.data_ptr(), scale.data_ptr(), ROWS, ld_x=8, ld_q=8)
    else:
        native.op_quant_q8(x.data_ptr(), native.DTYPE_BF16, ROWS, 1, q.data_ptr(), scale.data_ptr(), ld_x=8, ld_q=8)
    torch.cuda.synchronize()
    for i, r in enumerate(AT):
        want = 1 / 127 if norm else abs(x[r, 0].item()) / 127  # some of the multiples of 127 are rounded to 8 bits
        assert abs(scale[r].item() - want) <= 2.0 ** -24 * want and q[r].tolist() == [127 * (-1) ** i] + [3] * 7
        scale[r] = 0
        q[r, 0] = 0
    assert int(scale.count_nonzero()) == 0 and int(q.view(torch.int64).ne(0x0303030303030300).count_nonzero()) == 0


def test_append():
    """One buffer read as queries, keys and values; the last five rows stand at positions."""
    import torch
    rows = torch.zeros((ROWS, 16), dtype=torch.bfloat16, device="cuda")
    rows[-8:] = torch.randn((8, 16), device="cuda").to(torch.bfloat16)
    kc = torch.full((2, 1, 4, 16), 7.0, device="cuda")
    vc = kc.clone()
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, ROWS], dtype=torch.int32, device="cuda")
    kv = torch.tensor([5], dtype=torch.int32, device="cuda")
    native.KvAppend(1, 1, 16, 4, 2, 2, in_dtype=native.DTYPE_BF16, dtype=native.DTYPE_F32)(
        rows.data_ptr(), rows.data_ptr(), rows.data_ptr(), 0, kc.data_ptr(), vc.data_ptr(), table.data_ptr(), start.data_ptr(),
        kv.data_ptr(), 1, ROWS)
    torch.cuda.synchronize()
    for c in (kc, vc):
        got = torch.cat([c[1, 0], c[0, 0]])
        assert torch.equal(got[:5], rows[-5:].float()) and bool((got[5:] == 7).all())
