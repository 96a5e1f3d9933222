"""Attention over a shared prefix: the plan's tiles, the kernels against the definition in 64 bits, and the refusals.

Tolerances.  float32: dot products of hd terms, sums over the keys and the exponentials in 32 bits: (hd + keys + 64) roundings of 2^-24 at
worst in the sums, of the scores' absolute sums in the exponents; at random and for the scores of standard normal inputs used here
(sums of absolute terms up to some 60 in an exponent) 1e-5 of the values' size is many times what comes out.  bfloat16: a probability and the
result are rounded, half a step of 2^-9 .. 2^-8 each: an entry is off by at most 2^-8 of the largest value that it averages (the
probabilities' roundings, weighed by the probabilities) and 2^-8 of itself, and the sums as above (scores of bfloat16 inputs are exact
products, so the same 32-bit bound)."""
import copy

import pytest
import torch

import kernel_refs as ref
from tiny_inference_server_b200.kernels import ops
from tiny_inference_server_b200.kernels.attention_plan import SharedPrefixPlan


class Batch:
    """groups: (shared keys, [(keys of the request altogether, rows)]).  Slots are given out of order."""

    def __init__(self, groups, heads, kvh, hd, page, dtype=torch.bfloat16, seed=0, junk=float("nan"), spread=1.0):
        g = torch.Generator().manual_seed(seed)
        total = sum(len(r) for _, r in groups)
        self.heads, self.kvh, self.hd, self.page, self.dtype = heads, kvh, hd, page, dtype
        slots = torch.randperm(total + 2, generator=g)[:total].tolist()
        rnd = lambda *s: (torch.randn(*s, generator=g) * spread).to(dtype)  # noqa: E731
        most = max(n for _, r in groups for n, _ in r)
        width = -(-most // page) + 1
        table = torch.full((total + 2, width), -1, dtype=torch.int32)
        kvs, plan, positions, pages, i = [], [], [], 0, 0
        self.stored = []
        for shared, requests in groups:
            head, plan_r = rnd(shared, 2, kvh, hd), []
            full = shared // page
            shared_pages = list(range(pages, pages + full))
            pages += full
            for j in range(full):
                self.stored.append((shared_pages[j], j, head))
            for n, rows in requests:
                kv = torch.cat([head, rnd(n - shared, 2, kvh, hd)])
                mine = list(range(pages, pages + -(-n // page) - full))
                pages += len(mine)
                table[slots[i], : full + len(mine)] = torch.tensor(shared_pages + mine, dtype=torch.int32)
                for j, pg in enumerate(mine):
                    self.stored.append((pg, full + j, kv))
                kvs.append(kv)
                positions += list(range(n - rows, n))
                plan_r.append((slots[i], rows))
                i += 1
            plan.append((shared, plan_r))
        order = torch.randperm(pages + 1, generator=g)
        self.pages = pages + 1
        plane = torch.full((pages + 1, 2, kvh, page, hd), junk, dtype=dtype)
        for pg, index, kv in self.stored:
            lo = index * page
            part = kv[lo:lo + page]
            where = torch.arange(lo, lo + part.shape[0])
            for a in (0, 1):
                rows_ = torch.stack([ref.cache_row(part[r, a], int(where[r])) for r in range(part.shape[0])], 1)
                plane[order[pg], a, :, : part.shape[0]] = rows_
        table = torch.where(table >= 0, order[table.clamp(min=0).long()].int(), table)
        self.plan_groups, self.kvs = plan, kvs
        self.table, self.plane = table.cuda(), plane.cuda()
        self.positions = torch.tensor(positions, dtype=torch.int32).cuda()
        self.rows = len(positions)
        self.q = rnd(self.rows, heads * hd).cuda()
        self.fault = torch.zeros(4, dtype=torch.int32, device="cuda")
        self.plan = SharedPrefixPlan(plan, heads, kvh)

    def want(self, scale=None):
        """By the definition, in 64 bits; and the bound of a bfloat16 entry's error before its own rounding."""
        scale = self.hd ** -0.5 if scale is None else scale
        outs, sizes, row = [], [], 0
        g = self.heads // self.kvh
        pos = self.positions.tolist()
        q = self.q.double().reshape(self.rows, self.kvh, g, self.hd)
        i = 0
        for shared, requests in self.plan_groups:
            for _, rows in requests:
                kv = self.kvs[i].double().cuda()
                i += 1
                for _ in range(rows):
                    keys = pos[row] + 1
                    if keys <= shared:
                        outs.append(torch.zeros(self.heads * self.hd, dtype=torch.float64, device="cuda"))
                        sizes.append(outs[-1])
                    else:
                        s = torch.einsum("kgd,tkd->kgt", q[row], kv[:keys, 0]) * scale
                        p = torch.softmax(s, -1)
                        outs.append(torch.einsum("kgt,tkd->kgd", p, kv[:keys, 1]).reshape(-1))
                        sizes.append(torch.einsum("kgt,tkd->kgd", p, kv[:keys, 1].abs()).reshape(-1))
                    row += 1
        return torch.stack(outs), torch.stack(sizes)

    def run(self, out=None, **kw):
        out = torch.full((self.rows, self.heads * self.hd), 7.0, dtype=self.dtype, device="cuda") if out is None else out
        return ops.shared_prefix_attention(self.q, out, self.plane, self.table, self.positions, self.plan, self.fault, **kw)

    def check(self, got=None, scale=None, **kw):
        if got is None:
            got = self.run(scale=scale, **kw)[:, : self.heads * self.hd]
        want, size = self.want(scale)
        room = 1e-5 * (size + 1e-3)
        if self.dtype == torch.bfloat16:
            room += size * 2.0 ** -8 + want.abs() * 2.0 ** -8
        worst = ((got.double() - want).abs() - room).max().item()
        assert worst <= 0 and bool(torch.isfinite(got).all()), worst
        assert int(self.fault[0]) == 0
        return got


SHAPES = [  # groups, heads, kv heads, head size, page
    ([(0, [(1, 1)])], 1, 1, 16, 16),
    ([(0, [(5, 1), (70, 1)])], 4, 2, 32, 16),
    ([(16, [(17, 1)])], 3, 1, 64, 16),
    ([(16, [(17, 1), (40, 1)])], 12, 3, 128, 16),
    ([(100, [(101, 1), (130, 1), (164, 1)])], 8, 2, 64, 16),              # a shared page that is not full: each its own copy
    ([(64, [(70, 3), (65, 1), (200, 5)]), (33, [(40, 2)]), (0, [(9, 1)])], 6, 3, 64, 32),
    ([(1000, [(1003, 2)] * 9)], 32, 8, 128, 16),
    ([(700, [(701 + i, 1) for i in range(20)])], 24, 8, 64, 64),
    ([(300, [(310, 8), (333, 6)])], 8, 1, 96, 16),                        # rows of more heads than a tile has
    ([(257, [(300, 1), (258, 1)])], 33, 1, 48, 32),                       # 33 heads of one kv head
    ([(130, [(140, 1)] * 3)], 4, 4, 256, 16),
    ([(90, [(95, 2), (91, 1)])], 5, 5, 80, 1),                            # pages of one row
    ([(50, [(61, 2), (55, 1)])], 4, 2, 112, 7),                           # and of an odd number
    ([(128, [(129, 1)] * 40)], 8, 2, 128, 128),
    ([(2048, [(2049, 1), (3000, 1), (2500, 4)]), (512, [(600, 1)] * 5)], 16, 2, 128, 32),
    ([(15, [(16, 1), (20, 2)])], 4, 2, 64, 16),                           # less than a page is shared
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,heads,kvh,hd,page", SHAPES)
def test_against_the_definition(groups, heads, kvh, hd, page, dtype):
    Batch(groups, heads, kvh, hd, page, dtype, seed=hd + page).check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_as_paged_attention(dtype):
    """The framework's attention of the same rows, every request for itself."""
    b = Batch([(96, [(130, 1)] * 6), (0, [(33, 1)])], 8, 2, 64, 16, dtype, junk=0.0)
    got = b.check()
    slots = torch.tensor([s for _, r in b.plan_groups for s, _ in r], dtype=torch.int32, device="cuda")
    other = torch.empty_like(got)
    ops.paged_attention(b.q, other, b.plane, b.table, b.positions, slots, 8, 2, 64, 16, None, b.fault)
    b.check(other)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scale_strides_and_rows_behind(dtype):
    b = Batch([(64, [(70, 2), (90, 1)])], 4, 2, 64, 16, dtype)
    wide = torch.full((b.rows + 3, 4 * 64 + 128), 3.0, dtype=dtype, device="cuda")
    wide[: b.rows, :256] = b.q
    b.q = wide
    out = torch.full((b.rows + 3, 300), 7.0, dtype=dtype, device="cuda")
    b.run(out, scale=0.3, max_position=95)
    b.q = wide[: b.rows, :256]
    b.check(out[: b.rows, :256].contiguous(), scale=0.3)
    assert bool((out[b.rows:] == 7.0).all()) and bool((out[:, 256:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128, 96])
def test_rows_that_see_nothing(dtype, hd):
    """Padding rows, and rows inside the shared keys: zeros; the others as without them."""
    b = Batch([(64, [(70, 2), (90, 1), (65, 1)])], 4, 2, hd, 16, dtype)
    whole = b.check()
    b.positions[0], b.positions[3] = -1, 63
    got = b.check()
    assert bool((got[0] == 0).all()) and bool((got[3] == 0).all())
    assert torch.equal(got[1], whole[1]) and torch.equal(got[2], whole[2])
    b.positions.fill_(-5)
    assert bool((b.run() == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_later_row_that_is_not_finite_stays_with_those_that_see_it(dtype, hd, value):
    """Key and value of a drafted token are not finite: the rows before it are what they were."""
    b = Batch([(48, [(70, 4), (60, 2)])], 4, 2, hd, 16, dtype)
    whole = b.check()
    slot = b.plan_groups[0][1][0][0]
    page = int(b.table[slot, 68 // 16])
    b.plane[page, :, :, 68 % 16] = value
    got = b.run()
    same = [0, 1, 4, 5]
    assert torch.equal(got[same], whole[same])
    assert bool((~torch.isfinite(got[[2, 3]])).all())
    b.plane[page, 0, :, 68 % 16] = 0.0                              # the value alone
    got = b.run()
    assert torch.equal(got[same], whole[same]) and bool((~torch.isfinite(got[[2, 3]])).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores(dtype):
    """Scores of some hundreds: a softmax of almost one key, whatever part it is in."""
    b = Batch([(200, [(230, 1), (260, 2)])], 4, 2, 64, 16, dtype, spread=6.0)
    # float32 scores of size 36 * 64^0.5: their roundings (64 terms of up to 36 * 9, 2^-24 each, scaled) come out as up to 1e-3 of a probability
    want, size = b.want()
    got = b.run().double()
    assert ((got - want).abs() <= size * (2e-3 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) + want.abs() * 2.0 ** -8 + 1e-3).all()


@pytest.mark.gpu
def test_repeats_and_does_not_depend_on_the_others():
    groups = [(320, [(330, 1), (400, 1), (321, 3)])]
    b = Batch(groups, 8, 2, 128, 16)
    a = b.run()
    assert torch.equal(a, b.run())
    b.q[1] = 5.0
    c = b.run()
    assert torch.equal(a[0], c[0]) and torch.equal(a[2:], c[2:])


@pytest.mark.gpu
def test_growing_requests_captured():
    """A decode loop from one graph: positions move on the device, the plan stays."""
    b = Batch([(64, [(90, 1), (100, 1), (81, 1)])], 4, 2, 64, 16)
    out = torch.empty(b.rows, 4 * 64, dtype=torch.bfloat16, device="cuda")
    last = b.positions.clone()
    b.positions.copy_(last - 8)
    b.run(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(out)
    for back in (8, 3, 0):
        b.positions.copy_(last - back)
        out.zero_()
        graph.replay()
        b.check(out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = b.run()
    torch.cuda.current_stream().wait_stream(s)
    b.check(got)


@pytest.mark.gpu
def test_pages_that_are_not_there():
    for page in (-1, 10 ** 6):
        b = Batch([(32, [(40, 1), (50, 1)])], 4, 2, 64, 16, junk=0.0)
        b.table[b.plan_groups[0][1][1][0], 2] = page
        b.run()
        assert int(b.fault[0]) == 3
    b = Batch([(32, [(40, 1), (50, 1)])], 4, 2, 64, 16, junk=0.0)
    b.positions[1] = 10000                                          # behind the table's last page
    b.run()
    assert int(b.fault[0]) == 3


@pytest.mark.gpu
def test_long_cache_passes_32_bits():
    """Pages whose place in the pool takes more than 32 bits of elements."""
    b = Batch([(32, [(40, 1), (50, 1)])], 2, 1, 64, 16)
    whole = b.check()
    pages = (1 << 31) // (2 * 16 * 64) + 8
    plane = torch.zeros((pages + b.pages, 2, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
    plane[pages:] = b.plane
    b.plane = plane
    b.table = torch.where(b.table >= 0, b.table + pages, b.table)
    assert torch.equal(b.run(), whole)


def test_plan():
    plan = SharedPrefixPlan([(40, [(3, 1), (5, 7)]), (0, [(0, 2)])], 12, 4, "cpu")
    assert plan.rows == 10 and plan.max_slot == 5 and plan.max_shared == 40 and plan.min_shared == 0
    assert plan.own.tolist() == [[0, 3, 3, 40], [3, 16, 5, 40], [19, 5, 5, 40], [24, 6, 0, 0]]
    for size, tiles in plan.shared.items():
        assert [a + i for a, n, _, _ in tiles.tolist() for i in range(n)] == list(range(30))
        assert all(n <= size for _, n, _, _ in tiles.tolist())
    assert [x[2:] for x in plan.shared[64].tolist()] == [[3, 40], [0, 0]] and plan.most_heads == 24
    for groups, heads, kvh in (([], 4, 2), ([(0, [])], 4, 2), ([(-1, [(0, 1)])], 4, 2), ([(0, [(0, 0)])], 4, 2), ([(0, [(-1, 1)])], 4, 2),
                               ([(0, [(0, 1), (0, 1)])], 4, 2), ([(0, [(0, 1)])], 4, 3), ([(1 << 30, [(0, 1)])], 4, 2)):
        with pytest.raises(ValueError):
            SharedPrefixPlan(groups, heads, kvh, "cpu")


def test_refusals():
    plan = SharedPrefixPlan([(16, [(0, 1), (1, 1)])], 4, 2, "cpu")
    t = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    good = dict(q=bf(2, 128), out=bf(2, 128), plane=bf(3, 2, 2, 16, 32), block_table=t(2, 2), positions=t(2), plan=plan, fault=t(4))
    for bad in (dict(q=bf(1, 128)), dict(q=bf(2, 64)), dict(out=bf(1, 128)), dict(out=torch.zeros(2, 128)), dict(q=torch.zeros(2, 128)),
                dict(plane=bf(3, 2, 1, 16, 32)), dict(plane=bf(3, 2, 2, 16, 24)), dict(plane=bf(3, 2, 16, 32)), dict(plane=bf(3, 1, 2, 16, 32)),
                dict(plane=bf(3, 2, 2, 32, 16).transpose(3, 4)), dict(block_table=t(1, 2)), dict(block_table=t(2, 2).long()),
                dict(positions=t(1)), dict(positions=t(2).long()), dict(fault=torch.zeros(4)), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(q=bf(128, 2).t()), dict(q=bf(2, 129)), dict(q=bf(2, 129)[:, 1:]),
                dict(q=torch.zeros(2, 128).half(), out=torch.zeros(2, 128).half(), plane=torch.zeros(3, 2, 2, 16, 32).half())):
        with pytest.raises(ops.KernelError):
            ops.shared_prefix_attention(**{**good, **bad})
    with pytest.raises(ops.KernelError, match="own"):
        ops.shared_prefix_attention(**{**good, "out": good["q"]})
    with pytest.raises(ops.KernelError, match="CUDA tensors"):
        ops.shared_prefix_attention(**good)


@pytest.mark.gpu
def test_a_copy_of_a_plan():
    """A plan copied after a call reads its own tiles, not those it was copied from."""
    b = Batch([(32, [(40, 1), (50, 2)])], 4, 2, 64, 16)
    b.check()
    first, b.plan = b.plan, copy.deepcopy(b.plan)
    assert all(isinstance(x, (int, tuple)) for split in first.splits.values() for x in split) and len(first.splits) == 1
    first.own.zero_()
    for tiles in first.shared.values():
        tiles.zero_()
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("position", [1 << 20, 1 << 29, (1 << 31) - 1])
def test_a_position_far_behind_the_table(position, dtype):
    """Marked, and not walked to: the keys end where the tables do.  The other request's row is what it was."""
    b = Batch([(32, [(40, 1), (50, 1)])], 4, 2, 64, 16, dtype, junk=0.0)
    want = b.check()
    b.positions[1] = position
    for split in (dict(), dict(max_position=700)):                  # one own part, several
        b.fault.zero_()
        got = b.run(**split)
        assert int(b.fault[0]) == 3
        # (two results of other splits: each off by 2^-8 of itself and of the values' mean size, less than 2 here)
        room = 1e-5 * (want[0].abs() + 1) + (0 if dtype == torch.float32 else want[0].abs() * 2.0 ** -6 + 2.0 ** -6)
        assert bool(((got[0] - want[0]).abs() <= room).all())


def test_tables_shorter_than_the_shared_keys():
    plan = SharedPrefixPlan([(64, [(0, 1), (1, 1)])], 4, 2, "cpu")
    t = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    call = dict(q=bf(2, 128), out=bf(2, 128), plane=bf(3, 2, 2, 16, 32), positions=t(2), plan=plan, fault=t(4))
    with pytest.raises(ops.KernelError, match="64 shared keys"):
        ops.shared_prefix_attention(block_table=t(2, 3), **call)
    with pytest.raises(ops.KernelError, match="CUDA tensors"):
        ops.shared_prefix_attention(block_table=t(2, 4), **call)


def test_rows_of_the_result_on_one_another():
    plan = SharedPrefixPlan([(16, [(0, 1), (1, 1)])], 4, 2, "cpu")
    t = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ops.KernelError, match="on one another"):
        ops.shared_prefix_attention(q=bf(2, 128), out=bf(1, 128).expand(2, 128), plane=bf(3, 2, 2, 16, 32), block_table=t(2, 2), positions=t(2), plan=plan,
                                    fault=t(4))
