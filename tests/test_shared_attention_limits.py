"""What attention over a shared prefix refuses at the ends of the range."""
import ctypes

import pytest
import torch

from tiny_inference_server_b200.kernels import build, ops
from tiny_inference_server_b200.kernels.attention_plan import SharedPrefixPlan


def call(**other):
    t = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    plan = SharedPrefixPlan([(0, [(0, 1), (1, 1)])], 4, 2, "cpu")
    return ops.shared_prefix_attention(**{**dict(q=bf(2, 64), out=bf(2, 64), plane=bf(3, 2, 2, 16, 16), block_table=t(2, 2), positions=t(2), plan=plan, fault=t(4)),
                                          **other})


def test_pages_whose_keys_32_bits_do_not_count():
    """The loads look at pages up to 32 behind a row's last key: (last page + 32) times the page passes 2^31 for pages of more than 2^25 keys behind 2^30."""
    plane = lambda page: torch.empty((1, 2, 2, page, 16), dtype=torch.bfloat16, device="meta")  # noqa: E731
    for page in ((1 << 25) + 1, 1 << 27, 1 << 30):
        with pytest.raises(ops.KernelError, match="2\\^25 keys"):
            call(plane=plane(page))
    with pytest.raises(ops.KernelError, match="CUDA tensors"):
        call(plane=plane(1 << 25))


def test_the_launcher_refuses_them_too():
    lib = ctypes.CDLL(build.build_shared_attention(16))
    lib.tis_shared_attention.argtypes, lib.tis_last_error.restype = [ctypes.c_char_p], ctypes.c_char_p
    args = dict(zip("dtype q ldq out ldo plane table table_stride table_width num_pages positions own own_count wide wide_count wide_rows tensor own_parts shared_parts "
                    "rows H KVH page part_o part_ml fault stream most_heads own_heads".split(), [0] * 29))
    args.update(dtype=1, rows=1, H=1, KVH=1, page=(1 << 25) + 1, own_count=1, own_parts=1, wide_rows=16)
    assert lib.tis_shared_attention(ops._SHARED_ARGS.pack(*args.values(), 1.0)) != 0
    assert b"pages of" in lib.tis_last_error()
