"""A step of several samples of one prompt whose drafted tokens are verified, put together from the operators as a program would: 4-bit
products, keys and values written into the paged cache, attention over the shared prefix, the sampler's probabilities, the drafts' verification.
Against the same step in 64 bits, every stage from the stage before as the kernels left it."""
import pytest
import torch

import test_verify_drafts
from tiny_inference_server_b200.kernels import ops
from tiny_inference_server_b200.kernels.attention_plan import SharedPrefixPlan
from tiny_inference_server_b200.weights.w4 import pack_w4, quantize_w4, unpack_w4

pytestmark = pytest.mark.gpu

D, H, KVH, HD, PAGE, VOCAB = 256, 8, 2, 64, 16, 1000
SHARED, DRAFTS = 40, 2                                      # keys of the prompt (two whole pages), drafts of a request


def rotate(x, positions):
    """Half-split pairs, in 64 bits."""
    half = x.shape[-1] // 2
    angle = positions.double()[:, None, None] / 10000.0 ** (torch.arange(half, device=x.device).double() / half)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)


class Step:
    def __init__(self, dtype, requests=3, tail=(3, 9, 20)):
        g = torch.Generator().manual_seed(7)
        self.dtype, self.requests = dtype, requests
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        weights = {"qkv": rnd(D, (H + 2 * KVH) * HD) * D ** -0.5, "o": rnd(H * HD, D) * (H * HD) ** -0.5, "head": rnd(D, VOCAB) * 0.2}
        self.w = {k: pack_w4(*quantize_w4(v.cuda(), 64, True), 64) for k, v in weights.items()}
        self.dense = {k: unpack_w4(v, torch.float32).double() for k, v in self.w.items()}
        rows = DRAFTS + 1
        self.lens = [SHARED + t for t in tail]              # tokens in the cache before the step
        pages = [-(-(n + rows) // PAGE) for n in self.lens]
        table = torch.zeros((requests, max(pages)), dtype=torch.int32)
        free = torch.randperm(2 + sum(p - 2 for p in pages), generator=g).tolist()
        for r in range(requests):
            table[r, :2] = torch.tensor(free[:2])
            first = 2 + sum(p - 2 for p in pages[:r])
            table[r, 2:pages[r]] = torch.tensor(free[first:first + pages[r] - 2])
        self.table = table.cuda()
        self.plane = torch.zeros((len(free), 2, KVH, PAGE, HD), dtype=dtype, device="cuda")
        t = torch.arange(128, device="cuda").double()[:, None] / 10000.0 ** (torch.arange(HD // 2, device="cuda").double() / (HD // 2))
        self.cos, self.sin = t.cos().float(), t.sin().float()
        self.fault = torch.zeros(4, dtype=torch.int32, device="cuda")
        # the cache: the prompt once (request 0 writes it), each request's own tokens, as the framework writes them
        prompt = rnd(SHARED, (H + 2 * KVH) * HD)
        self.kv = []
        for r, n in enumerate(self.lens):
            qkv = torch.cat([prompt, rnd(n - SHARED, (H + 2 * KVH) * HD)]).to(dtype).cuda()
            self.kv.append(qkv.double())
            self._write(qkv.clone(), torch.arange(n), torch.full((n,), r))
        self.positions = torch.tensor([n + j for n in self.lens for j in range(rows)], dtype=torch.int32, device="cuda")
        self.slots = torch.tensor([r for r in range(requests) for _ in range(rows)], dtype=torch.int32, device="cuda")
        self.plan = SharedPrefixPlan([(SHARED, [(r, rows) for r in range(requests)])], H, KVH)
        n = requests * rows
        self.x = rnd(n, D).to(dtype).cuda()
        self.drafts = torch.randint(0, VOCAB, (requests, DRAFTS), generator=g).int().cuda()
        self.u = torch.rand(requests, rows, generator=g).cuda()
        self.room = {"qkv": torch.empty(n, (H + 2 * KVH) * HD, dtype=dtype, device="cuda"), "heads": torch.empty(n, H * HD, dtype=dtype, device="cuda"),
                     "o": torch.empty(n, D, dtype=dtype, device="cuda"), "logits": torch.empty(n, VOCAB, device="cuda"),
                     "probs": torch.empty(n, VOCAB, device="cuda"), "drawn": torch.empty(n, dtype=torch.int32, device="cuda"),
                     "tokens": torch.empty(requests, rows, dtype=torch.int32, device="cuda"), "kept": torch.empty(requests, dtype=torch.int32, device="cuda")}
        self.settings = (torch.full((n,), 0.8, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda"),
                         torch.ones(n, device="cuda"), None, None, torch.zeros(n, dtype=torch.int64, device="cuda"), torch.arange(n, device="cuda"))

    def _write(self, qkv, positions, slots):
        ops.rope_kv_write(qkv, positions.int().cuda(), slots.int().cuda(), self.cos, self.sin, self.plane, self.table, H, KVH, HD, PAGE, self.fault)

    def run(self):
        m = self.room
        ops.gemm_w4(self.x, self.w["qkv"], m["qkv"])
        ops.rope_kv_write(m["qkv"], self.positions, self.slots, self.cos, self.sin, self.plane, self.table, H, KVH, HD, PAGE, self.fault)
        ops.shared_prefix_attention(m["qkv"], m["heads"], self.plane, self.table, self.positions, self.plan, self.fault, max_position=127)
        ops.gemm_w4(m["heads"], self.w["o"], m["o"])
        m["o"].add_(self.x)
        logits = ops.gemm_w4(m["o"], self.w["head"])
        m["logits"].copy_(logits)
        ops.sample_rows(m["logits"], *self.settings, m["drawn"], m["probs"])
        ops.verify_drafts(m["probs"].view(self.requests, DRAFTS + 1, VOCAB), None, self.drafts, self.u, None, m["tokens"], m["kept"])

    def check(self):
        """Every stage against 64 bits.  half: the rounding of a stored entry; float32 sums as in the operators' own tests, bounded here by 1e-5
        of the absolute sums; float32 rotations have angles to 2^-24 * 128."""
        half = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -24
        m, x = self.room, self.x.double()
        qkv = x @ self.dense["qkv"]
        size = x.abs() @ self.dense["qkv"].abs()
        n, hq = x.shape[0], H * HD
        q = rotate(qkv[:, :hq].view(n, H, HD), self.positions).reshape(n, hq)
        # a rotation mixes two entries that were rounded to the type, and rounds again
        room = 2e-5 * size[:, :hq].view(n, H, HD).amax(-1, keepdim=True) + 3 * half * qkv[:, :hq].view(n, H, HD).abs().amax(-1, keepdim=True)
        got = m["qkv"][:, :hq].double().view(n, H, HD)
        assert ((got - q.view(n, H, HD)).abs() <= room).all()
        # attention from the queries that the kernel had and the keys that were written (rounded after the rotation)
        at = 0
        for r, length in enumerate(self.lens):
            rows = DRAFTS + 1
            new = torch.cat([torch.zeros(rows, hq, dtype=torch.float64, device="cuda"), m["qkv"][at:at + rows, hq:].double()], 1)
            kv = torch.cat([self.kv[r], new])
            k = rotate(kv[:, hq:hq + KVH * HD].view(-1, KVH, HD), torch.arange(length + rows, device="cuda")).to(self.dtype).double()
            v = kv[:, hq + KVH * HD:].view(-1, KVH, HD)
            for j in range(rows):
                s = torch.einsum("kgd,tkd->kgt", m["qkv"][at + j, :hq].double().view(KVH, H // KVH, HD), k[: length + j + 1]) * HD ** -0.5
                p = torch.softmax(s, -1)
                o = torch.einsum("kgt,tkd->kgd", p, v[: length + j + 1])
                size = torch.einsum("kgt,tkd->kgd", p, v[: length + j + 1].abs())
                # probabilities and results rounded, keys by half a step more where the angles' 32 bits turned a rounding (scores of a few units)
                assert ((m["heads"][at + j].double().view_as(o) - o).abs() <= size * (2 * half + 1e-4) + o.abs() * half + 1e-6).all()
            at += rows
        o = m["heads"].double() @ self.dense["o"]
        size = m["heads"].double().abs() @ self.dense["o"].abs()
        assert ((m["o"].double() - o - x).abs() <= 1e-5 * size + half * o.abs() + half * (o + x).abs() + 1e-6).all()
        logits = m["o"].double() @ self.dense["head"]
        size = m["o"].double().abs() @ self.dense["head"].abs()
        assert ((m["logits"].double() - logits).abs() <= 1e-5 * size + half * logits.abs() + 1e-6).all()
        probs = torch.softmax(m["logits"].double() / 0.8, -1)
        assert ((m["probs"].double() - probs).abs() <= 1e-5 * probs + 1e-7).all()
        want, kept = test_verify_drafts.plain(m["probs"].view(self.requests, -1, VOCAB).cpu(), None, self.drafts.cpu(), self.u.cpu())
        assert m["tokens"].cpu().tolist() == want.tolist() and m["kept"].cpu().tolist() == kept.tolist()
        assert int(self.fault[0]) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(dtype):
    s = Step(dtype)
    s.run()
    s.check()
    # drafts that the target is sure of are kept: the arg-max of every place, and numbers near zero
    s.drafts.copy_(s.room["logits"].view(s.requests, DRAFTS + 1, VOCAB)[:, :DRAFTS].argmax(-1).int())
    s.u[:, :DRAFTS] = 1e-6
    s.run()
    s.check()
    assert s.room["kept"].tolist() == [DRAFTS] * s.requests


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_replayed(dtype):
    s = Step(dtype)
    s.run()
    first = {k: v.clone() for k, v in s.room.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for v in s.room.values():
        v.zero_()
    graph.replay()
    assert all(torch.equal(s.room[k], v) for k, v in first.items() if k != "drawn")
    s.x.copy_(torch.randn(s.x.shape, generator=torch.Generator().manual_seed(1)))
    s.u.copy_(torch.rand(s.u.shape, generator=torch.Generator().manual_seed(2)))
    graph.replay()
    s.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_at_once(dtype):
    """Two steps of their own on two streams: neither's scratch is the other's."""
    a, b = Step(dtype), Step(dtype, 2, (1, 15))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, step in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                step.run()
    torch.cuda.synchronize()
    a.check()
    b.check()
