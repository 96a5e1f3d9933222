"""Results of products and of attention that reach into the rows they are made of: refused; beside them in one buffer: taken."""
import pytest
import torch

from test_shared_attention_limits import call
from test_w4 import make
from tiny_inference_server_b200.kernels import ops
from tiny_inference_server_b200.weights.w4 import pack_w4


def test_rows_meet_as_their_bytes_do():
    g = torch.Generator().manual_seed(0)
    seen = set()
    for _ in range(4000):
        rows, wide_a, wide_b, gap = (int(torch.randint(1, 6, (1,), generator=g)) for _ in range(4))
        ld = max(wide_a, wide_b) + gap
        a, b = (int(torch.randint(0, 40, (1,), generator=g)) for _ in range(2))
        places = [{x + r * ld + c for r in range(-rows, 2 * rows) for c in range(w)} if all_rows else {x + r * ld + c for r in range(rows) for c in range(w)}
                  for x, w, all_rows in ((a, wide_a, True), (b, wide_b, False), (a, wide_a, False))]
        meet = ops._rows_meet(4 * a, ld, wide_a, 4 * b, ld, wide_b, rows, 4)
        if places[1] & places[2]:
            assert meet
        elif not places[1] & places[0]:                         # (nor would they if the first had more rows)
            assert not meet
        seen.add(meet)
    assert seen == {False, True}
    assert not ops._rows_meet(0, 8, 8, 0, 8, 8, 0, 4) and ops._rows_meet(0, 0, 8, 28, 8, 8, 5, 4) and not ops._rows_meet(0, 0, 8, 32, 8, 8, 5, 4)


def test_products():
    w = pack_w4(*make(32, 16, 32, False), 32)
    room = torch.zeros(1000, dtype=torch.bfloat16)
    at = lambda first, cols, ld=64, n=3: room.as_strided((n, cols), (ld, 1), first)  # noqa: E731
    x = at(0, 32)
    for out in (at(16, 16), at(31, 16), at(64, 16), at(60, 16, 64), at(20, 16, 16), at(130, 16, 16), at(144, 16, 100)):
        with pytest.raises(ops.KernelError, match="where the rows are"):
            ops.gemm_w4(x, w, out)
    with pytest.raises(ops.KernelError, match="where the rows are"):
        ops.gemm_w4(room[:32].expand(3, 32), w, at(30, 16))
    for out in (at(32, 16), at(48, 16), at(160, 16, 16), at(192, 16), at(500, 16, 100)):
        with pytest.raises(ops.KernelError, match="CUDA tensors"):
            ops.gemm_w4(x, w, out)


def test_attention():
    room = torch.zeros(1000, dtype=torch.bfloat16)
    at = lambda first, ld=256: room.as_strided((2, 64), (ld, 1), first)  # noqa: E731
    for out in (at(0), at(8), at(56), at(256), at(248), at(40, 64)):
        with pytest.raises(ops.KernelError, match="own"):
            call(q=at(0), out=out)
    for out in (at(64), at(192), at(512), at(320, 64)):
        with pytest.raises(ops.KernelError, match="CUDA tensors"):
            call(q=at(0), out=out)
