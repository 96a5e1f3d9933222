"""What products with weights of four bits refuse, and what they take at the ends of the range."""
import dataclasses

import pytest
import torch

from test_w4 import dense, kernel, make  # noqa: F401
from tiny_inference_server_b200.kernels import ops
from tiny_inference_server_b200.weights.w4 import pack_w4, quantize_w4


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


@pytest.mark.parametrize("zeros", [False, True])
def test_weights_that_have_no_scale(zeros):
    """One NaN or infinity took its group's other weights with it."""
    for value in (float("nan"), float("inf"), -float("inf")):
        w = torch.randn(70, 5, generator=torch.Generator().manual_seed(0))
        w[66, 2] = value
        with pytest.raises(ValueError, match="not finite"):
            quantize_w4(w, 32, zeros)
    with pytest.raises(ValueError, match="not finite"):
        quantize_w4(torch.full((4, 4), 1e300, dtype=torch.float64), 32, zeros)
    # the largest numbers of both signs: a range of twice the largest, in steps that are finite
    most = torch.finfo(torch.float32).max
    w = torch.tensor([[most], [-most], [0.0], [most / 2]])
    codes, scales, z = quantize_w4(w, 32, zeros)
    assert bool(torch.isfinite(scales.float()).all())
    at = codes.double() - (z.double() if zeros else 8.0)
    # half a step, one more half for the zero point, and the scale's rounding (2^-8) over up to 15 steps
    assert bool(((at * scales.double() - w.double()).abs() <= scales.double() * (1.0 + 15 * 2.0 ** -8)).all())


@pytest.mark.gpu
def test_packed_weights_in_one_buffer(kernel):  # noqa: F811
    w = pack_w4(*make(300, 80, 32, True, device="cuda"), 32)
    other = dataclasses.replace(w, words=behind(w.words, 16), scales=behind(w.scales, 4), zeros=behind(w.zeros, 2))
    x = torch.randn(5, 300, device="cuda").bfloat16()
    assert torch.equal(ops.gemm_w4(x, other), ops.gemm_w4(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-100, -110, -118, -125, -130, -140])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows", [1, 3, 8])
def test_very_small_float32_rows_keep_their_bits(exponent, zeros, rows, kernel):  # noqa: F811
    """Entries whose last bits lie far below bfloat16's smallest number, and entries below float32's smallest normal one.  Room: that of test_w4.py, and what
    is rounded to steps of 2^-149, by half of one each: a group's scaled sum of the high parts (8 groups), the same of the two lower parts (2^-8 of it) and
    their two joins."""
    g = torch.Generator().manual_seed(rows)
    codes, scales, z = make(256, 70, 32, zeros, 7, "cuda")
    x = (torch.randn(rows, 256, generator=g, dtype=torch.float64) * 2.0 ** exponent).float().cuda()
    d = dense(codes, scales, z, 32)
    want, size = x.double() @ d, x.double().abs() @ d.abs()
    got = ops.gemm_w4(x, pack_w4(codes, scales, z, 32)).double()
    room = (24 * 2.0 ** -23 + 4 * 2.0 ** -24) * size + (8 + 2 * 8 * 2.0 ** -8 + 2) * 2.0 ** -150
    assert ((got - want).abs() <= room).all(), ((got - want).abs() / size).max().item()


@pytest.mark.gpu
def test_float32_rows_up_to_the_largest(kernel):  # noqa: F811
    """Every bit of numbers of any size counts, the largest float32 number's too."""
    codes, scales, _ = make(64, 16, 64, False, 6, "cuda")
    codes.fill_(8)
    codes[:5] = 9
    scales.fill_(1.0)
    w = pack_w4(codes, scales, None, 64)
    x = torch.zeros(5, 64, device="cuda")
    for i, v in enumerate((torch.finfo(torch.float32).max, 1 + 2.0 ** -23, 2.0 ** -126 * (1 + 2.0 ** -23), 2.0 ** -149, 2.0 ** -127 + 2.0 ** -149)):
        x[i, i] = v
    got = ops.gemm_w4(x, w)
    assert torch.equal(got, x.sum(1, keepdim=True).expand_as(got))


@pytest.mark.gpu
def test_packed_weights_are_there_when_they_are_returned():
    """A product's kernel reads weights ahead of the wait for the kernel in front of it: none that packs may still run."""
    codes = torch.full((4096, 65536), 3, dtype=torch.uint8, device="cuda")      # milliseconds of work
    scales, z = torch.ones(128, 65536, device="cuda").bfloat16(), codes[:128].clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pack_w4(codes, scales, z, 32)
        assert s.query()
