"""Which kernel a four-bit product goes to: what the mma.sync launcher holds in one piece, at every edge, and the choice made of it."""
import ctypes

import pytest

from tiny_inference_server_b200.kernels import build, ops


@pytest.fixture
def library(monkeypatch):
    lib = ctypes.CDLL(build.build())
    monkeypatch.setattr(ops, "_lib", lib)
    ops._w4_tensor.cache_clear()
    yield lib
    ops._w4_tensor.cache_clear()


def bytes_of(eights, k, n):
    """Shared memory of a CTA with x in one piece: staged rows of whole turns of eight warps, 16 entries behind each, and two tiles' sums of all warps, in floats."""
    whole = -(-k // 512) * 512
    columns = 32 if eights == 2 or (eights == 1 and n > 296 * 16) else 16
    return eights * 8 * (whole + 16) * 2 + 2 * 8 * eights * 8 * (columns + 1) * 4


@pytest.mark.parametrize("staged", [1, 8, 9, 16, 17, 24])
@pytest.mark.parametrize("n", [1, 2304, 4736, 4737, 28672, 131072])
def test_one_piece_at_every_edge(staged, n, library):
    eights, last = -(-staged // 8), None
    for k in range(1, 9000):
        fits = bool(library.tis_gemm_w4_one_piece(staged, k, n))
        assert fits == (bytes_of(eights, k, n) <= 112 * 1024), k
        assert last in (None, fits) or (last and not fits)         # a single edge
        if last and not fits:
            edge = k - 1
        last = fits
    assert edge == {1: 6144 if n <= 4736 else 5632, 2: 2048, 3: 1536}[eights]


def test_in_several_pieces_only_where_that_was_measured_faster(library):
    for staged in range(1, 25):
        for k in (100, 1536, 1537, 2048, 2049, 2240, 2560, 3392, 4096, 5632, 5633, 6144, 6145, 6848, 6849, 20000):
            for n in (16, 2304, 4096, 8192, 16384, 18944, 18945, 28672, 37888, 37889, 131072):
                for group in (32, 64, 128, 4096):
                    tensor, one = ops._w4_tensor(staged, k, n, group), library.tis_gemm_w4_one_piece(staged, k, n)
                    if not one and not tensor:
                        assert staged <= 16 and n > 148 * 128 and (group == 32 or n <= 296 * 128)
                    if one and tensor:
                        assert group >= 64 and n > 96 * 128 and staged > 8
    assert ops._w4_tensor(25, 64, 16, 32)


@pytest.mark.parametrize("staged,k,n", [(16, 2560, 4096), (9, 2560, 2304), (24, 2048, 8192), (17, 2048, 28672), (8, 6144, 8192), (1, 6656, 2304)])
def test_between_the_sizes_that_fit(staged, k, n, library):
    """x that does not fit in one piece, of products of ordinary width: three times as long in several pieces."""
    assert all(ops._w4_tensor(staged, k, n, group) for group in (32, 64, 128))


@pytest.mark.parametrize("staged,k,n", [(1, 1536, 2304), (8, 4096, 28672), (8, 4096, 4096), (9, 2005, 5501), (16, 2048, 2304), (24, 1536, 2304)])
def test_sizes_that_fit(staged, k, n, library):
    assert not any(ops._w4_tensor(staged, k, n, group) for group in (32, 64, 128))


@pytest.mark.parametrize("dtype,rows", [(1, 25), (0, 9), (1, 64)])
def test_the_mma_launcher_refuses_more_rows_than_it_is_built_for(dtype, rows, library):
    library.tis_last_error.restype = ctypes.c_char_p
    library.tis_gemm_w4.argtypes = [ctypes.c_char_p]
    assert library.tis_gemm_w4(ops._W4_ARGS.pack(dtype, 0, 64, 0, 0, 0, 0, 64, rows, 64, 64, 32, 0, 0, 0, 0)) != 0
    assert b"rows" in library.tis_last_error()
