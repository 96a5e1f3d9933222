"""Products with weights of four bits: the layout of the codes, and the kernel against the definition in 64 bits.

Tolerances.  The kernel's weights are exact, x is exact (float32 as three bfloat16 numbers), a product of both is exact in 32 bits.
What is rounded is the sums: a chunk of 64 products in 32 bits by the tensor cores, which may cut the last bit of every operand
of an addition instead of rounding it (2^-23 relative, 17 terms at a time, 4 times, and a scale): each partial result is off by at most some
(17 + 4 + 2) 2^-23 of the sum of the absolute terms, and the sum over the chunks adds one 2^-24 of the running sum each.  So |error| <=
(24 * 2^-23 + chunks * 2^-24) * sum |x| |w| bounds every entry, and a bfloat16 result adds half a step, 2^-8 of itself."""
import copy
import dataclasses
import pickle

import pytest
import torch

from tiny_inference_server_b200.kernels import ops
from tiny_inference_server_b200.weights.w4 import pack_w4, quantize_w4, unpack_w4


def make(k, n, group, zeros, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8)
    scales = (torch.rand(groups, n, generator=g) * 0.02 + 0.001).bfloat16()
    z = torch.randint(0, 16, (groups, n), generator=g, dtype=torch.uint8) if zeros else None
    return codes.to(device), scales.to(device), None if z is None else z.to(device)


def dense(codes, scales, zeros, group):
    at = torch.arange(codes.shape[0], device=codes.device) // group
    return (codes.double() - (zeros.double()[at] if zeros is not None else 8.0)) * scales.double()[at]


def check(x, codes, scales, zeros, group, out=None):
    w = pack_w4(codes, scales, zeros, group)
    got = ops.gemm_w4(x, w, out)
    d = dense(codes, scales, zeros, group)
    want = x.double() @ d
    room = (24 * 2.0 ** -23 + -(-x.shape[1] // 64) * 2.0 ** -24) * (x.double().abs() @ d.abs())
    if x.dtype == torch.bfloat16:
        room += want.abs() * 2.0 ** -8 + 2.0 ** -133
    assert got.shape == want.shape and got.dtype == x.dtype
    worst = ((got.double() - want).abs() - room).max().item()
    assert worst <= 0, worst
    return got


@pytest.mark.parametrize("k,n,group", [(64, 16, 32), (128, 32, 128), (1, 1, 32), (205, 51, 32), (333, 17, 64), (100, 40, 4096)])
@pytest.mark.parametrize("zeros", [False, True])
def test_pack_and_back(k, n, group, zeros):
    codes, scales, z = make(k, n, group, zeros)
    w = pack_w4(codes, scales, z, group)
    assert w.shape == (k, n) and w.words.numel() * 8 == -(-k // 64) * 64 * -(-n // 128) * 128
    assert torch.equal(unpack_w4(w, torch.float32).double(), dense(codes, scales, z, group))


def test_words_of_a_lane():
    """The documented place of every code."""
    codes, scales, _ = make(128, 176, 64, False)
    w = pack_w4(codes, scales, None, 64)
    for strip, chunk, lane, word in ((0, 0, 0, 0), (1, 1, 13, 3), (2, 0, 31, 2), (10, 1, 6, 1)):
        g, t = lane // 4, lane % 4
        k0, c = 64 * chunk + 16 * word + 4 * t, 16 * strip + g
        want = [codes[k0, c], codes[k0, c + 8], codes[k0 + 2, c], codes[k0 + 2, c + 8],
                codes[k0 + 1, c], codes[k0 + 1, c + 8], codes[k0 + 3, c], codes[k0 + 3, c + 8]]
        v = int(w.words[strip // 8, chunk, strip % 8, lane, word])
        assert [(v >> (4 * i)) & 15 for i in range(8)] == [int(x) for x in want]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_is_within_half_a_step(zeros, dtype):
    w = torch.randn(300, 40, generator=torch.Generator().manual_seed(1)).to(dtype)
    w[:64, 3] = 0.0
    w[64:128, 4] = w[64:128, 4].abs() + 1.0                     # (all of one sign)
    codes, scales, z = quantize_w4(w, 64, zeros)
    back = unpack_w4(pack_w4(codes, scales, z, 64), torch.float32)
    at = torch.arange(300) // 64
    # half a step; the scale is rounded to bfloat16 (2^-8), which the largest code, 15 steps from the zero point, feels at most
    room = scales.float()[at] * (0.5 + 15 * 2.0 ** -8) * 1.001
    if zeros:
        room = room + scales.float()[at] * 0.5                  # (the zero point is a whole code)
    assert bool(((w.float() - back).abs() <= room).all())
    assert bool((back[:64, 3] == 0).all())


def test_refusals():
    codes, scales, z = make(128, 32, 64, True)
    for bad in ((codes.int(), scales, z, 64), (codes, scales.float(), z, 64), (codes, scales, z, 48), (codes, scales, z, 16),
                (codes, scales[:1], z, 64), (codes, scales, z[:, :5], 64), (codes, scales, z.int(), 64), (codes + 10, scales, z, 64),
                (codes, scales, z + 15, 64), (codes[0], scales, z, 64), (codes[:0], scales[:0], None, 64)):
        with pytest.raises(ValueError):
            pack_w4(*bad)
    for bad in (torch.zeros(3), torch.zeros(3, 3, dtype=torch.int32), torch.zeros(0, 3)):
        with pytest.raises(ValueError):
            quantize_w4(bad)
    w = pack_w4(codes, scales, z, 64)
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    for a, out in ((x[:, :64], None), (x.half(), None), (x.t().contiguous().t(), None), (x, torch.zeros(2, 32)),
                   (x, torch.zeros(2, 31, dtype=torch.bfloat16)), (x, torch.zeros(32, 2, dtype=torch.bfloat16).t())):
        with pytest.raises(ops.KernelError):
            ops.gemm_w4(a, w, out)
    square = pack_w4(*make(32, 32, 32, False), 32)
    y = torch.zeros(2, 32, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="where the rows are"):
        ops.gemm_w4(y, square, y)
    with pytest.raises(ops.KernelError, match="CUDA tensors"):
        ops.gemm_w4(x, w)
    for change in (dict(words=w.words[:, :1]), dict(scales=w.scales.float()), dict(zeros=w.zeros.transpose(0, 1)), dict(n=200), dict(k=129), dict(group=32),
                   dict(words=w.words.transpose(3, 4).contiguous().transpose(3, 4))):
        with pytest.raises(ValueError):
            dataclasses.replace(w, **change)


SIZES = [(1, 1, 1, 32), (1, 64, 16, 32), (1, 1536, 2304, 128), (8, 1536, 520, 64), (5, 2005, 1001, 32), (3, 96, 33, 64), (9, 512, 160, 128),
         (17, 1000, 100, 128), (27, 777, 64, 32), (40, 4096, 256, 64), (64, 2048, 320, 128), (64, 9000, 48, 32), (65, 300, 40, 32),
         (200, 640, 72, 256), (2, 20000, 16, 64), (7, 4096, 20000, 128), (33, 130, 19000, 32), (60, 8200, 24, 16384)]


@pytest.fixture(params=[None, False, True], ids=["chosen", "mma", "tcgen05"])
def kernel(request, monkeypatch):
    monkeypatch.setattr(ops, "W4_TENSOR", request.param)
    yield
    if torch.cuda.is_available():
        assert int(ops.tc_fault()[0].item()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n,group", SIZES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products(rows, k, n, group, zeros, dtype, kernel):
    codes, scales, z = make(k, n, group, zeros, rows + k + n, "cuda")
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).to(dtype).cuda()
    check(x, codes, scales, z, group)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_and_what_lies_beside_them(dtype, kernel):
    codes, scales, z = make(512, 80, 64, True, 3, "cuda")
    for offset, extra in ((0, 0), (8, 8), (1, 3), (4, 4)):
        room = torch.full((6, 512 + offset + extra), float("nan"), dtype=dtype, device="cuda")
        x = room[:, offset:offset + 512]
        x.copy_(torch.randn(6, 512, generator=torch.Generator().manual_seed(offset)))
        wide = torch.full((8, 100), 7.0, dtype=dtype, device="cuda")
        check(x, codes, scales, z, 64, wide[1:7, 5:85])
        wide[1:7, 5:85] = 7.0
        assert bool((wide == 7.0).all())                        # nothing else was written
    row = torch.randn(1, 512, device="cuda").to(dtype)
    check(row.expand(5, 512), codes, scales, z, 64)             # one row for all


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_numbers_far_apart_and_none(dtype, kernel):
    """Large beside small, infinities and NaN: what is not finite stays in its row."""
    codes, scales, z = make(256, 48, 32, True, 5, "cuda")
    x = torch.randn(6, 256, generator=torch.Generator().manual_seed(1)) * torch.logspace(-18, 18, 256)[None]
    x[1, 7], x[2, 100], x[3, 255] = float("inf"), float("nan"), -float("inf")
    x = x.to(dtype).cuda()
    w = pack_w4(codes, scales, z, 32)
    got = ops.gemm_w4(x, w).double()
    d = dense(codes, scales, z, 32)
    for r in (0, 4, 5):
        check(x[r:r + 1], codes, scales, z, 32)
        assert torch.equal(got[r:r + 1], ops.gemm_w4(x[r:r + 1], w).double())
    assert bool(got[2].isnan().all())
    for r, k in ((1, 7), (3, 255)):
        hit = d[k] != 0
        assert torch.equal(got[r][hit], (x[r, k].double() * d[k])[hit]) and bool(got[r][~hit].isnan().all())
    tiny = torch.full((2, 256), 2.0 ** -126, device="cuda").to(dtype)
    want = tiny.double() @ d
    # entries of 2^-126 times weights: results of 2^-126 and below, in steps of 2^-149 (bfloat16 2^-133); the lower parts of a float are zero here
    assert ((ops.gemm_w4(tiny, w).double() - want).abs() <= want.abs() * 2.0 ** -8 + (2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -140)).all()


@pytest.mark.gpu
def test_float32_rows_keep_their_bits(kernel):
    """A float's low bits count: x and the same less its last sixteen bits differ by what they are."""
    codes, scales, z = make(128, 16, 128, False, 6, "cuda")
    codes.fill_(9)
    scales.fill_(1.0)
    x = torch.zeros(1, 128, device="cuda")
    x[0, 5] = 1.0 + 2.0 ** -23
    assert ops.gemm_w4(x, pack_w4(codes, scales, None, 128))[0, 3].item() == 1.0 + 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 24, 48])
def test_a_row_does_not_depend_on_the_others_and_runs_repeat(rows, kernel):
    codes, scales, z = make(1024, 400, 64, True, 8, "cuda")
    w = pack_w4(codes, scales, z, 64)
    x = torch.randn(rows, 1024, device="cuda").bfloat16()
    a = ops.gemm_w4(x, w)
    assert torch.equal(a, ops.gemm_w4(x, w))
    y = x.clone()
    y[1:] = float("nan")
    assert torch.equal(a[0], ops.gemm_w4(y, w)[0])


@pytest.mark.gpu
def test_streams_and_graphs(kernel):
    codes, scales, z = make(1536, 640, 128, False, 9, "cuda")
    w = pack_w4(codes, scales, z, 128)
    x = torch.randn(4, 1536, device="cuda").bfloat16()
    want = ops.gemm_w4(x, w)
    out, other = torch.zeros_like(want), torch.zeros_like(want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.gemm_w4(x, w, out)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_w4(x, w, out)
        ops.gemm_w4(out[:, :0].new_zeros(0, 1536), w)           # no rows: nothing is launched
        ops.gemm_w4(x, w, other)
    x.copy_(torch.randn(4, 1536, device="cuda"))
    graph.replay()
    want = ops.gemm_w4(x, w)
    assert torch.equal(out, want) and torch.equal(other, want)


@pytest.mark.gpu
def test_quantized_matrix_like_the_unpacked_one():
    g = torch.Generator().manual_seed(4)
    m = (torch.randn(768, 300, generator=g) * 0.02).cuda()
    w = pack_w4(*quantize_w4(m, 64, True), 64)
    x = torch.randn(10, 768, generator=g).cuda()
    got, d = ops.gemm_w4(x, w).double(), unpack_w4(w, torch.float32).double()
    # (unpacked weights are rounded to float32, 2^-24 each)
    room = (24 * 2.0 ** -23 + 12 * 2.0 ** -24 + 2.0 ** -24) * (x.double().abs() @ d.abs())
    assert ((got - x.double() @ d).abs() <= room).all()


def test_packed_weights_hold_tensors_and_sizes_only():
    """Nothing of a place in memory: copies, and weights read from a file, have places of their own."""
    w = pack_w4(*make(100, 40, 32, True), 32)
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert set(vars(other)) == {f.name for f in dataclasses.fields(w)} == {"words", "scales", "zeros", "k", "n", "group"}
        assert torch.equal(other.words, w.words) and other.words.data_ptr() != w.words.data_ptr()


@pytest.mark.gpu
def test_a_copy_of_packed_weights(kernel):
    w = pack_w4(*make(512, 96, 64, True, device="cuda"), 64)
    x = torch.randn(3, 512, device="cuda").bfloat16()
    want = ops.gemm_w4(x, w)
    other = copy.deepcopy(w)
    for part in (w.words, w.scales, w.zeros):
        part.zero_()
    assert torch.equal(ops.gemm_w4(x, other), want)


def test_rows_of_the_result_on_one_another():
    w = pack_w4(*make(64, 32, 32, False), 32)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    for out in (torch.zeros(1, 32, dtype=torch.bfloat16).expand(3, 32), torch.zeros(200, dtype=torch.bfloat16).as_strided((3, 32), (16, 1))):
        with pytest.raises(ops.KernelError, match="on one another"):
            ops.gemm_w4(x, w, out)
