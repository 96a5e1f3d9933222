"""Products with weights of four bits where a CTA takes several tiles of columns: sums, operands, zero points and rounds carried from one to the
next.  Tolerances: those of test_w4.py."""
import pytest
import torch

from test_w4 import check, make
from tiny_inference_server_b200.kernels import ops

pytestmark = pytest.mark.gpu


# more than 2 x 296 tiles of 128 columns, the last of them not full; an odd and an even number of chunks, one alone, a last group that is not full
@pytest.mark.parametrize("k", [40, 300, 640, 704])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,dtype", [(5, torch.bfloat16), (40, torch.bfloat16), (64, torch.bfloat16), (3, torch.float32), (21, torch.float32)])
def test_three_tiles_a_cta(k, group, zeros, rows, dtype, monkeypatch):
    monkeypatch.setattr(ops, "W4_TENSOR", True)
    n = 2 * 296 * 128 + 1000
    codes, scales, z = make(k, n, group, zeros, k + rows, "cuda")
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).to(dtype).cuda()
    got = check(x, codes, scales, z, group)
    assert torch.equal(got, check(x, codes, scales, z, group))
    assert int(ops.tc_fault()[0].item()) == 0


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("rows,dtype", [(1, torch.bfloat16), (8, torch.bfloat16), (16, torch.bfloat16), (24, torch.bfloat16), (2, torch.float32), (8, torch.float32)])
def test_tiles_of_few_columns(group, rows, dtype, monkeypatch):
    """The mma.sync kernel: tiles of 16 or 32 columns, three and more a CTA."""
    monkeypatch.setattr(ops, "W4_TENSOR", False)
    codes, scales, z = make(333, 30001, group, True, rows, "cuda")
    x = torch.randn(rows, 333, generator=torch.Generator().manual_seed(rows)).to(dtype).cuda()
    check(x, codes, scales, z, group)
