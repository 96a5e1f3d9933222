"""Attention over a shared prefix where the kernels' loops go round: shared tiles on the tcgen05 kernel with several tiles of 128 keys a part, of both
head sizes and all pages that it takes, and more own tiles than CTAs.  Tolerances: those of test_shared_attention.py, which hold for any number of keys."""
import pytest
import torch

import kernel_refs as ref
from test_shared_attention import Batch
from tiny_inference_server_b200.kernels import ops

pytestmark = pytest.mark.gpu


@pytest.fixture
def tensor(monkeypatch):
    """Shared keys to the tcgen05 kernel whatever the number of row heads."""
    monkeypatch.setattr(ops, "SHARED_TC_HEADS", 0)


def split(monkeypatch, shared, own=1):
    """Parts of the shared and of the own keys."""
    monkeypatch.setattr(ops, "_split_parts", lambda items, tiles, resident, start, join=0.0, most=64: min(tiles, shared if start == 4 else own))


def takes_tensor(b):
    (_, _, wide, (_, _, tensor, _, parts)), = b.plan.splits.values()
    assert tensor and wide == 128
    return parts


# one to nine tiles of 128 keys, the last of 128, of 16 and of 112; parts of an even and an odd number of tiles, and empty ones
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("shared,parts", [(128, 1), (250, 1), (520, 1), (1030, 1), (1150, 2), (1040, 3), (1152, 4), (1152, 7)])
def test_several_tiles_a_part(hd, page, shared, parts, tensor, monkeypatch):
    split(monkeypatch, parts)
    b = Batch([(shared, [(shared + 1, 1), (shared + 30, 3), (shared + 70, 2)])], 12, 3, hd, page, seed=shared + hd)
    first = b.check()
    assert takes_tensor(b) == min(parts, -(-(shared // page * page) // 128))
    assert all(torch.equal(first, b.run()) for _ in range(5))


@pytest.mark.parametrize("hd", [64, 128])
def test_groups_of_different_lengths(hd, tensor, monkeypatch):
    """More row heads than a tile has, a group without shared keys, one with less than a page of them, parts that end before others."""
    split(monkeypatch, 3, 2)
    b = Batch([(900, [(910 + i, 2) for i in range(9)]), (0, [(40, 1)]), (300, [(301, 1)] * 3), (9, [(30, 2)])], 16, 2, hd, 16, seed=hd)
    b.check()
    takes_tensor(b)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("parts", [1, 2])
def test_large_scores_raise_the_maximum(hd, parts, tensor, monkeypatch):
    """Scores of some hundreds over eight tiles: sums and outputs are rescaled on the way."""
    split(monkeypatch, parts)
    b = Batch([(1024, [(1030, 1), (1060, 2)])], 8, 2, hd, 16, spread=6.0, seed=hd)
    want, size = b.want()
    got = b.run().double()
    takes_tensor(b)
    # as test_large_scores: the scores' 32-bit roundings come out as up to 1e-3 of a probability, twice that for twice the terms
    assert ((got - want).abs() <= size * (2e-3 * hd / 64 + 2.0 ** -8) + want.abs() * 2.0 ** -8 + 1e-3).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("parts", [1, 3])
def test_rows_that_see_nothing(hd, parts, tensor, monkeypatch):
    """Padding rows, warps and requests without any other: zeros; the others as without them."""
    split(monkeypatch, parts)
    b = Batch([(640, [(650, 5), (660, 30), (641, 1)])], 4, 2, hd, 16)      # 72 row heads a kv head: three warps, the last not full
    whole = b.check()
    takes_tensor(b)
    b.positions[0], b.positions[3] = -1, 639
    b.positions[6:34] = -1                                                  # a warp of the softmax and more
    got = b.run()
    gone = [0, 3, *range(6, 34)]
    rest = [r for r in range(b.rows) if r not in gone]
    assert bool((got[gone] == 0).all()) and torch.equal(got[rest], whole[rest])
    b.positions.fill_(-5)
    assert bool((b.run() == 0).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_values_that_are_not_finite(hd, value, tensor, monkeypatch):
    """In an own key: the rows that see it, and no others.  In a shared one: its group's rows, and no others."""
    split(monkeypatch, 2)
    b = Batch([(512, [(540, 4), (530, 2)]), (256, [(300, 2)])], 4, 2, hd, 16)
    whole = b.check()
    takes_tensor(b)
    slot = b.plan_groups[0][1][0][0]
    page = int(b.table[slot, 538 // 16])
    b.plane[page, :, :, 538 % 16] = value
    got = b.run()
    same = [0, 1, 4, 5, 6, 7]
    assert torch.equal(got[same], whole[same]) and bool((~torch.isfinite(got[[2, 3]])).all())
    b.plane[int(b.table[slot, 200 // 16]), 1, :, 200 % 16] = value
    got = b.run()
    assert torch.equal(got[6:], whole[6:]) and bool((~torch.isfinite(got[:6])).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_repeats_and_does_not_depend_on_the_others(hd, tensor, monkeypatch):
    split(monkeypatch, 2)
    b = Batch([(700, [(710, 1), (800, 1), (701, 3)] * 4)], 8, 2, hd, 16)
    a = b.check()
    takes_tensor(b)
    assert all(torch.equal(a, b.run()) for _ in range(20))
    b.q[1] = 5.0
    c = b.run()
    assert torch.equal(a[0], c[0]) and torch.equal(a[2:], c[2:])


@pytest.mark.parametrize("hd", [64, 128])
def test_captured(hd, tensor, monkeypatch):
    """Positions move on the device between replays, and another capture of the same plan has scratch of its own."""
    split(monkeypatch, 2)
    b = Batch([(600, [(690, 1), (700, 2)])], 12, 2, hd, 32)
    out, other = (torch.empty(b.rows, 12 * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    last = b.positions.clone()
    b.run(out)
    takes_tensor(b)
    graphs = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    for graph, to in zip(graphs, (out, other)):
        with torch.cuda.graph(graph):
            b.run(to)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for back in (60, 3, 0):
        b.positions.copy_(last - back)
        out.zero_()
        other.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        b.check(out)
        assert torch.equal(out, other)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,own", [(64, 1), (64, 3), (128, 1), (128, 2), (256, 1)])
def test_more_own_tiles_than_ctas(hd, own, dtype, monkeypatch):
    """100 requests of 8 kv heads: 800 and more items for 296 CTAs (148 of heads of 256).  Of different lengths, some with padding rows, some
    with nothing else."""
    split(monkeypatch, 2, own)
    g = torch.Generator().manual_seed(own)
    lens = torch.randint(1, 150, (100,), generator=g).tolist()
    b = Batch([(40, [(40 + n, 1 + i % 3 if n > 3 else 1) for i, n in enumerate(lens[:70])]), (0, [(n, 1) for n in lens[70:]])], 8, 8, hd, 16, dtype, seed=hd)
    assert b.plan.own.shape[0] * 8 * own > 2 * 296
    whole = b.check()
    assert all(torch.equal(whole, b.run()) for _ in range(5))
    gone = torch.arange(0, b.rows, 7).tolist() + list(range(20, 30))
    for r in gone:
        b.positions[r] = -1
    rest = [r for r in range(b.rows) if r not in gone]
    got = b.run()
    assert bool((got[gone] == 0).all()) and torch.equal(got[rest], whole[rest])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shared,page", [(1040, 16), (1152, 64), (64, 64), (992, 32)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_an_infinity_in_the_last_shared_page(hd, shared, page, value, tensor, monkeypatch):
    """A value that every row sees with a positive weight: infinite there, finite in all other columns, whatever lies behind the last shared key in its tile."""
    split(monkeypatch, 1)
    b = Batch([(shared, [(shared + 3, 1), (shared + 40, 2)])], 4, 2, hd, page)
    whole = b.check()
    takes_tensor(b)
    slot = b.plan_groups[0][1][0][0]
    key = shared - 1
    row = b.plane[int(b.table[slot, key // page]), 1, 0, key % page]
    column = int(ref.cache_row(torch.arange(hd).bfloat16(), key)[5])
    row[5] = value
    got = b.run().view(b.rows, 4, hd)
    assert bool((got[:, :2, column] == value).all())
    rest = [c for c in range(hd) if c != column]
    assert torch.equal(got[:, :, rest], whole.view(b.rows, 4, hd)[:, :, rest]) and torch.equal(got[:, 2:], whole.view(b.rows, 4, hd)[:, 2:])
