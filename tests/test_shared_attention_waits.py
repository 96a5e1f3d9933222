"""The requests' own keys wait for the kernel of the shared ones, however long that takes: kernels built here whose bounded waits end after some 0.1 ms, and
shared keys that take longer."""
import ctypes
import subprocess

import pytest
import torch

from tiny_inference_server_b200.kernels import build, ops
from tiny_inference_server_b200.kernels.attention_plan import SharedPrefixPlan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("waits") / "shared.so")
    files = [f"{build.CSRC}/{f}" for f in (*build.PER_HEAD_SIZE_SHARED, "errors.cu")]
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-DTIS_HD=16", "-DTIS_MBAR_SPINS=64", "-I", build.CSRC, "-shared", "-o", out, *files], check=True)
    lib = ctypes.CDLL(out)
    lib.tis_last_error.restype, lib.tis_shared_attention.argtypes = ctypes.c_char_p, [ctypes.c_char_p]
    lib.widest = lib.tis_shared_attn_widest()
    return lib


def test_shared_keys_that_take_longer_than_a_wait(impatient, monkeypatch):
    heads, page, requests, rows, prefix = 16, 16, 160, 8, 1 << 17
    full = prefix // page
    g = torch.Generator(device="cuda").manual_seed(0)
    plane = torch.randn((full + 2 * requests, 2, 1, page, 16), generator=g, device="cuda").bfloat16()
    table = torch.cat([torch.arange(full).expand(requests, full), full + torch.arange(2 * requests).view(requests, 2)], 1).int().cuda()
    positions = (prefix + 10 + torch.arange(rows)).repeat(requests).int().cuda()
    q = torch.randn((requests * rows, heads * 16), generator=g, device="cuda").bfloat16()
    plan = SharedPrefixPlan([(prefix, [(i, rows) for i in range(requests)])], heads, 1)
    assert plan.own.shape[0] > 3 * 296                          # own tiles: more than three a CTA, of which two are ahead
    fault = torch.zeros(4, dtype=torch.int32, device="cuda")

    def run():
        return ops.shared_prefix_attention(q, torch.zeros_like(q), plane, table, positions, plan, fault, max_position=prefix + 31)

    want = run()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    again = run()
    b.record()
    b.synchronize()
    assert a.elapsed_time(b) > 0.5 and torch.equal(again, want)  # ms
    ((_, _, _, (_, _, _, own_parts, _)),) = plan.splits.values()
    assert own_parts == 1                                       # joined by the own tiles themselves
    monkeypatch.setitem(ops._shared_attn_libs, 16, impatient)
    for _ in range(3):
        assert torch.equal(run(), want) and int(fault[0]) == 0
