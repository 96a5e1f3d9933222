"""Verification of drafted tokens: the kernel against the rule written request by request in 64 bits, and its refusals.

Whole numbers have to be equal.  Both sides add up a row in 64 bits, in another order: the sums agree to some 1e-15 of
themselves, so a number drawn at random from 2^24 would have to lie that near the edge of a token for the tokens to differ."""
import numpy as np
import pytest
import torch

from tiny_inference_server_b200.kernels import ops


def plain(p, q, drafts, u, lens=None):
    p, drafts, u = p.double().numpy(), drafts.numpy(), u.double().numpy()
    q = None if q is None else q.double().numpy()
    n, k1, v = p.shape

    def mass(row):
        return np.where((row > 0) & (row < np.inf), row, 0.0)

    tokens, accepted = np.full((n, k1), -1, np.int64), np.zeros(n, np.int64)
    for b in range(n):
        most = k1 - 1 if lens is None else min(max(int(lens[b]), 0), k1 - 1)
        a = 0
        while a < most:
            d = drafts[b, a]
            if not 0 <= d < v:
                break
            if not u[b, a] * (1.0 if q is None else mass(q[b, a])[d]) < mass(p[b, a])[d]:
                break
            a += 1
        row = left = mass(p[b, a])
        if a < most:
            if q is not None:
                left = np.maximum(row - mass(q[b, a]), 0.0)
            elif 0 <= drafts[b, a] < v:
                left = row.copy()
                left[drafts[b, a]] = 0.0
            if not left.sum() > 0:
                left = row
        sums = np.cumsum(left)
        beyond = np.nonzero(sums > u[b, -1] * sums[-1])[0]
        some = np.nonzero(left)[0]
        tokens[b, :a] = drafts[b, :a]
        tokens[b, a] = beyond[0] if len(beyond) else (some[-1] if len(some) else -1)
        accepted[b] = a
    return torch.from_numpy(tokens).int(), torch.from_numpy(accepted).int()


def make(n, k, v, seed, sharp=3.0, near=1.0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(n, k + 1, v, generator=g) * sharp
    p = logits.softmax(-1)
    q = (logits[:, :k] + near * torch.randn(n, k, v, generator=g)).softmax(-1)
    drafts = torch.multinomial(q.reshape(n * k, v), 1, generator=g).reshape(n, k).int() if k else torch.zeros(n, 0, dtype=torch.int32)
    return p, q, drafts, torch.rand(n, k + 1, generator=g)


def check(p, q, drafts, u, lens=None, place=lambda t: t):
    tokens, accepted = ops.verify_drafts(place(p.cuda()), None if q is None else place(q.cuda()), drafts.cuda(), u.cuda(),
                                         None if lens is None else lens.cuda())
    want, kept = plain(p, q, drafts, u, lens)
    assert accepted.cpu().tolist() == kept.tolist()
    assert tokens.cpu().tolist() == want.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,v", [(1, 4, 32000), (1, 0, 1), (3, 2, 1), (5, 3, 2), (4, 1, 3), (7, 2, 127), (9, 5, 129), (70, 31, 50),
                                   (13, 5, 1000), (6, 3, 8193), (2, 7, 50001), (33, 4, 4096), (1, 1, 131072), (1, 8, 131075),
                                   (700, 3, 211), (3, 1, 1048579)])
@pytest.mark.parametrize("distribution", [True, False])
def test_tokens(n, k, v, distribution):
    p, q, drafts, u = make(n, k, v, n + k + v)
    if not distribution:
        drafts = p[:, :k].argmax(-1).int()
    check(p, q if distribution else None, drafts, u)


@pytest.mark.gpu
@pytest.mark.parametrize("distribution", [True, False])
def test_ragged_and_odd_drafts(distribution):
    n, k, v = 40, 6, 777
    p, q, drafts, u = make(n, k, v, 5, near=0.3)
    lens = torch.randint(-1, k + 3, (n,), generator=torch.Generator().manual_seed(1)).int()     # held between 0 and k
    drafts[3, 0], drafts[4, 1], drafts[5, 2], drafts[6, 5] = -1, v, 2 ** 31 - 1, -2 ** 31
    check(p, q if distribution else None, drafts, u, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strided_rows(offset):
    """Rows of every alignment: a longer row, a shifted start, requests behind one another in another order."""
    p, q, drafts, u = make(6, 3, 4099, 11)

    def place(t):
        room = torch.full((t.shape[1], t.shape[0], t.shape[2] + 5 + offset), 7.0, device="cuda")
        view = room.transpose(0, 1)[:, :, offset:offset + t.shape[2]]
        view.copy_(t)
        return view

    check(p, q, drafts, u, place=place)
    row = p[:1, :1].expand(6, 4, 4099)                        # one row for all
    tokens, accepted = ops.verify_drafts(row[:1, :1].cuda().expand(6, 4, 4099), q.cuda(), drafts.cuda(), u.cuda())
    want, kept = plain(row, q, drafts, u)
    assert tokens.cpu().tolist() == want.tolist() and accepted.cpu().tolist() == kept.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("v", [5, 300, 40000])
def test_edges_of_the_draw(v):
    """The smallest and largest numbers, rows of one entry, of none, p equal to q, and entries that are no probabilities."""
    n, k = 12, 2
    p, q, drafts, u = make(n, k, v, v)
    u[:, -1] = torch.tensor([0.0, 1 - 2.0 ** -24, 2.0 ** -149, 0.5] * 3)
    u[:4, 0] = 1 - 2.0 ** -24
    p[0], p[1] = 0.0, 0.0
    p[1, :, v - 1] = 1.0                                      # all mass at the end
    p[2], p[3] = 0.0, 0.0
    p[3, :, 0] = 1e-40                                        # subnormal
    q[4:6] = p[4:6, :k]                                       # nothing left of the difference
    u[4:6, 0] = 1.0                                           # (not below one: equal probabilities refuse)
    p[6, :, v // 2], p[6, :, 1], p[7, :, 2] = float("nan"), float("inf"), -1.0
    q[6, :, 0], q[7, :, 3], q[8, :, 4] = float("nan"), float("inf"), float("-inf")
    p[9], q[10] = float("nan"), 0.0
    u[11] = 1.0                                               # beyond the range: the last entry with mass
    check(p, q, drafts, u)
    check(p, None, drafts, u)


@pytest.mark.gpu
def test_dyadic_rows_meet_the_edges_exactly():
    """Equal entries and numbers that are multiples of them: a running sum equal to the number is not beyond it."""
    v, k = 4096, 1
    p = torch.full((64, k + 1, v), 1.0 / v)
    q = torch.full((64, k, v), 2.0 / v)
    q[:, :, 1::2] = 0.0
    drafts = torch.zeros(64, k, dtype=torch.int32)
    u = torch.zeros(64, k + 1)
    u[:, 0] = 0.75
    u[:, 1] = torch.arange(64) / 64.0
    check(p, q, drafts, u)
    assert ops.verify_drafts(p.cuda(), q.cuda(), drafts.cuda(), u.cuda())[0][32, 0].item() == 2049


@pytest.mark.gpu
def test_long_strides_pass_32_bits():
    """Rows that lie further apart than 32 bits of elements count."""
    v, k = 40, 1
    step = (1 << 31) + 64
    room = torch.empty(step + v, dtype=torch.float32, device="cuda")
    view = room.as_strided((1, 2, v), (0, step, 1))
    p, q, drafts, u = make(1, k, v, 3, near=0.0)
    view.copy_(p)
    u[0, 0] = 0.0
    tokens, accepted = ops.verify_drafts(view, q.cuda(), drafts.cuda(), u.cuda())
    want, kept = plain(p, q, drafts, u)
    assert kept.item() == 1 and tokens.cpu().tolist() == want.tolist() and accepted.item() == 1


@pytest.mark.gpu
def test_captured_streams_and_results_given():
    p, q, drafts, u = [t.cuda() for t in make(20, 4, 5000, 8)]
    want, kept = ops.verify_drafts(p, q, drafts, u)
    tokens, accepted = torch.full((20, 5), 99, dtype=torch.int32, device="cuda"), torch.full((20,), 99, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.verify_drafts(p, q, drafts, u, None, tokens, accepted)
    torch.cuda.current_stream().wait_stream(s)
    assert got[0] is tokens and torch.equal(tokens, want) and torch.equal(accepted, kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(p, q, drafts, u, None, tokens, accepted)
    other = [t.cuda() for t in make(20, 4, 5000, 9)]
    for mine, new in zip((p, q, drafts, u), other):
        mine.copy_(new)
    graph.replay()
    want, kept = ops.verify_drafts(*other)
    assert torch.equal(tokens, want) and torch.equal(accepted, kept)


@pytest.mark.gpu
def test_probabilities_of_the_sampler():
    """The sampler's own probabilities as the target's: top-k leaves most tokens none, a greedy row one."""
    n, k, v = 3, 2, 1000
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(n * (k + 1), v, generator=g).cuda()
    rows = n * (k + 1)
    p = torch.empty(rows, v, device="cuda")
    temps = torch.tensor([1.0, 0.0, 0.7] * 3, device="cuda")
    ops.sample_rows(logits, temps, torch.full((rows,), 20, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda"),
                    torch.ones(rows, device="cuda"), None, None, torch.zeros(rows, dtype=torch.int64, device="cuda"),
                    torch.arange(rows, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda"), p)
    drafts = logits.reshape(n, k + 1, v)[:, :k].argmax(-1).int()
    u = torch.rand(n, k + 1, generator=g)
    tokens, accepted = ops.verify_drafts(p.reshape(n, k + 1, v), None, drafts, u.cuda())
    want, kept = plain(p.reshape(n, k + 1, v).cpu(), None, drafts.cpu(), u)
    assert tokens.cpu().tolist() == want.tolist() and accepted.cpu().tolist() == kept.tolist()


@pytest.mark.gpu
def test_chances():
    """Many numbers for one request: kept with chance sum min(p, q), and the token that comes out is the target's."""
    n, v = 40000, 8
    p, q, _, _ = make(1, 1, v, 4, sharp=1.0)
    g = torch.Generator().manual_seed(5)
    drafts = torch.multinomial(q.reshape(1, v).expand(n, v), 1, generator=g).int()
    tokens, accepted = ops.verify_drafts(p.cuda().expand(n, 2, v), q.cuda().expand(n, 1, v), drafts.cuda(), torch.rand(n, 2, generator=g).cuda())
    share = torch.minimum(p[0, 0], q[0, 0]).sum().item()
    # five standard deviations of a share of n draws, at most 0.5 / sqrt(n) each
    assert abs(accepted.float().mean().item() - share) < 2.5 / n ** 0.5
    counts = torch.bincount(tokens[:, 0].cpu().long(), minlength=v) / n
    assert (counts - p[0, 0]).abs().max().item() < 2.5 / n ** 0.5


def test_refusals():
    p, q, drafts, u = make(3, 2, 10, 0)
    good = dict(target_probs=p, draft_probs=q, drafts=drafts, uniforms=u)
    for bad in (dict(target_probs=p.double()), dict(draft_probs=q.double()), dict(drafts=drafts.long()), dict(uniforms=u.double()),
                dict(draft_probs=q[:, :1]), dict(draft_probs=q[..., :9]), dict(drafts=drafts[:, :1]), dict(uniforms=u[:, :2]),
                dict(target_probs=p.transpose(1, 2).contiguous().transpose(1, 2)), dict(draft_lens=torch.zeros(2, dtype=torch.int32)),
                dict(draft_lens=torch.zeros(3)), dict(tokens=torch.zeros(3, 2, dtype=torch.int32)), dict(accepted=torch.zeros(3)),
                dict(drafts=drafts.t().contiguous().t()), dict(tokens=torch.zeros(3, 3)),
                dict(target_probs=torch.zeros(1, 33, 4), draft_probs=None, drafts=torch.zeros(1, 32, dtype=torch.int32), uniforms=torch.zeros(1, 33))):
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(**{**good, **bad})
    with pytest.raises(ops.KernelError, match="CUDA tensors"):
        ops.verify_drafts(**good)


def test_tokens_in_the_place_of_an_argument():
    p, q, drafts, u = make(3, 2, 10, 0)
    room = torch.zeros(20, dtype=torch.int32)
    room[:6] = drafts.reshape(-1)
    for bad in (dict(drafts=room[:6].view(3, 2), tokens=room[:9].view(3, 3)), dict(tokens=u.view(torch.int32)),
                dict(tokens=room[:9].view(3, 3), accepted=room[:3])):
        with pytest.raises(ops.KernelError, match="do not lie where"):
            ops.verify_drafts(**{**dict(target_probs=p, draft_probs=q, drafts=drafts, uniforms=u), **bad})


@pytest.mark.gpu
def test_kept_drafts_in_the_place_of_their_lengths():
    """A request's length is read before its result is written."""
    p, q, drafts, u = (t.cuda() for t in make(40, 3, 5000, 3))
    lens = (torch.arange(40, dtype=torch.int32) % 4).cuda()
    tokens, kept = ops.verify_drafts(p, q, drafts, u, lens)
    there = lens.clone()
    again, place = ops.verify_drafts(p, q, drafts, u, there, accepted=there)
    assert place.data_ptr() == there.data_ptr() and torch.equal(again, tokens) and torch.equal(there, kept)
