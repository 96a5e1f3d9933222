"""What products with weights of four bits refuse, and what they take at the ends of the range."""
import dataclasses

import pytest
import torch

from test_w4 import dense, kernel, make  # noqa: F401
from tiny_inference_server_b200.kernels import ops
from tiny_inference_server_b200.weights.w4 import pack_w4


def behind(x, offset):
    """A copy of x that starts ``offset`` bytes behind a place of 64."""
    room = torch.zeros(x.numel() * x.element_size() + 128, dtype=torch.uint8, device=x.device)
    first = -room.data_ptr() % 64 + offset
    view = room[first:first + x.numel() * x.element_size()].view(x.dtype).view(x.shape)
    view.copy_(x)
    return view


def test_packed_weights_off_their_places():
    """Contiguous parts of one buffer that the kernels' loads could not read."""
    w = pack_w4(*make(128, 48, 64, True), 64)
    for name, offsets, good in (("words", (4, 8, 12, 20), (16, 32)), ("scales", (2, 6), (4, 8)), ("zeros", (1, 3), (2, 6))):
        for offset in offsets:
            with pytest.raises(ValueError, match=f"{name}: starts on"):
                dataclasses.replace(w, **{name: behind(getattr(w, name), offset)})
        for offset in good:
            assert torch.equal(getattr(dataclasses.replace(w, **{name: behind(getattr(w, name), offset)}), name), getattr(w, name))


@pytest.mark.gpu
def test_packed_weights_in_one_buffer(kernel):  # noqa: F811
    w = pack_w4(*make(300, 80, 32, True, device="cuda"), 32)
    other = dataclasses.replace(w, words=behind(w.words, 16), scales=behind(w.scales, 4), zeros=behind(w.zeros, 2))
    x = torch.randn(5, 300, device="cuda").bfloat16()
    assert torch.equal(ops.gemm_w4(x, other), ops.gemm_w4(x, w))
