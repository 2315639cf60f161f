"""Attention of one new token of every sequence where groups of sequences share their first keys, against 64 bits.

Bounds (u: unit roundoff of the 16-bit type, 2^-8 bf16, 2^-11 fp16; e4m3 caches are read in fp16).  A weight is rounded to 16 bits as an operand (u sum w|v|) and
stands against a sum of unrounded ones, the output is rounded once; a logit is an fp32 sum of head_dim products, (head_dim + 16) 2^-23 of sum |q k|
scale off at most, which moves a weight by as much; fp16 weights below the normal range lose up to 2^-30 of the largest each, and an fp16
output is 2^-25 off where it is subnormal.
"""

import math

import pytest
import torch

from fms_model_optimizer_b200 import ops
from oracle import attention as OA

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
F8 = torch.float8_e4m3fn


class Case:
    """`groups`: (prefix, lengths) pairs, lengths with the prefix counted in.  Pages are scattered, whatever no sequence has is NaN, and table entries that are not to be
    read are no pages at all."""

    def __init__(self, seed, dev, groups, hq, hkv, dim, page, dtype, f8=False, std=1.5):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.dtype, self.page, self.hq, self.hkv, self.dim, self.groups = dev, dtype, page, hq, hkv, dim, groups
        self.lens = [n for _, ns in groups for n in ns]
        self.prefix = [p for p, ns in groups for _ in ns]
        b = len(self.lens)
        wide = max(1, max(-(-p // page) for p, _ in groups))
        per = max(1, max([-(-n // page) for n in self.lens] + [1]))
        own = [range(min(p, n) // page, -(-n // page)) if n > p else range(0) for p, n in zip(self.prefix, self.lens)]
        pages = sum(-(-p // page) for p, _ in groups) + sum(len(r) for r in own) + 3
        order = iter(torch.randperm(pages, generator=g).tolist())
        self.prefix_table = torch.full((len(groups), wide), 1 << 30, dtype=torch.int32)
        self.table = torch.full((b, per), -(1 << 30), dtype=torch.int32)
        ct = F8 if f8 else dtype
        k, v = (torch.full((pages, hkv, page, dim), math.nan) for _ in range(2))
        for i, (p, _) in enumerate(groups):
            for j in range(-(-p // page)):
                at = next(order)
                self.prefix_table[i, j] = at
                for t in (k, v):
                    t[at, :, : min(page, p - j * page)] = torch.randn(hkv, min(page, p - j * page), dim, generator=g)
        for i, r in enumerate(own):
            for j in r:
                at = next(order)
                self.table[i, j] = at
                lo, hi = max(self.prefix[i] - j * page, 0), min(page, self.lens[i] - j * page)
                for t in (k, v):
                    t[at, :, lo:hi] = torch.randn(hkv, hi - lo, dim, generator=g)
        self.k, self.v = k.to(ct), v.to(ct)
        self.ks, self.vs = (torch.rand(hkv, generator=g) * 0.5 + 0.75 if f8 else None for _ in range(2))
        self.q = (torch.randn(b, hq, dim, generator=g) * std).to(dtype)
        self.at = torch.tensor([0] + torch.tensor([len(ns) for _, ns in groups]).cumsum(0).tolist(), dtype=torch.int32)

    def args(self):
        lens = torch.tensor(self.lens, dtype=torch.int32)
        prefix = torch.tensor([p for p, _ in self.groups], dtype=torch.int32)
        return [t.to(self.dev) for t in (self.q, self.k, self.v, self.prefix_table, prefix, self.at, self.table, lens)]

    def scales(self):
        return dict(k_scale=self.ks.to(self.dev), v_scale=self.vs.to(self.dev)) if self.ks is not None else {}

    def place(self, b, key):
        """(page, offset) of a key of sequence b."""
        group = int(torch.searchsorted(self.at, b, right=True)) - 1
        table = self.prefix_table[group] if key < self.prefix[b] else self.table[b]
        return int(table[key // self.page]), key % self.page

    def check(self, got, window=0, sinks=0, scale=None):
        got = got.cpu()
        for b, n in enumerate(self.lens):
            where = [self.place(b, j) for j in range(n)]
            pages, offsets = (torch.tensor([w[i] for w in where], dtype=torch.long) for i in (0, 1))
            for h in range(self.hkv):
                heads = slice(h * self.hq // self.hkv, (h + 1) * self.hq // self.hkv)
                kk, vv = (x.float()[pages, h, offsets].double().view(n, self.dim) * (1.0 if s is None else s[h].double()) for x, s in ((self.k, self.ks), (self.v, self.vs)))
                want, weighted, size = OA.attend(self.q[b, heads], kk, vv, n - 1, window, sinks, scale or self.dim**-0.5)
                wt = torch.float16 if self.ks is not None else self.dtype
                logits = 2 * (self.dim + 16) * 2.0**-23 * size[:, None] + 2.0**-20
                tol = (2 * U[wt] + logits) * weighted + U[self.dtype] * want.abs() + 1e-30
                if wt == torch.float16:
                    tol = tol + n * 2.0**-30 * (float(vv.abs().max()) if n else 0.0) + 2.0**-25
                err = (got[b, heads].double() - want).abs()
                assert bool((err <= tol).all()), (b, h, n, float((err - tol).max()), float(err.max()))


SHAPES = [
    ([(16, [17])], 1, 1, 64, 16, 0, 0), ([(300, [301, 350, 420]), (40, [41, 44])], 8, 2, 128, 16, 0, 0), ([(2048, [2049 + 31 * i for i in range(4)])], 32, 8, 128, 64, 0, 0),
    ([(129, [130] * 20)], 5, 1, 96, 24, 0, 0), ([(1000, [1400, 1100, 1001]), (0, [5, 700]), (77, [78])], 4, 4, 64, 7, 100, 3), ([(513, [520, 4000])], 40, 4, 128, 128, 128, 130),
    ([(700, [0, 701, 3, 0, 700, 1200]), (64, [64, 0])], 12, 12, 64, 33, 0, 0), ([(64, [0, 0]), (50, [60])], 4, 2, 16, 5, 0, 0), ([(900, [901 + i for i in range(40)])], 24, 1, 128, 48, 0, 0),
    ([(500, [505, 900, 760]), (500, [501] * 9)], 9, 1, 64, 16, 450, 4), ([(1, [2, 3]), (2, [3])], 2, 1, 48, 1, 1, 0), ([(0, [40, 0, 3])], 8, 2, 64, 16, 0, 0),
    ([(640, [650 + 3 * i for i in range(70)])], 8, 2, 64, 32, 0, 0), ([(3000, [3001 + 7 * i for i in range(36)]), (2500, [2501 + i for i in range(33)])], 8, 1, 128, 64, 0, 0)]  # fmt: skip


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("groups,hq,hkv,dim,page,window,sinks", SHAPES)
def test_against_64_bits(cuda_dev, dtype, f8, groups, hq, hkv, dim, page, window, sinks):
    c = Case(len(groups) + dim + hq, cuda_dev, groups, hq, hkv, dim, page, dtype, f8)
    args = c.args()
    got = ops.prefix_attention(*args, window=window, sinks=sinks, **c.scales())
    ops.check_status(cuda_dev)
    assert torch.equal(got, ops.prefix_attention(*args, window=window, sinks=sinks, **c.scales())), "two runs differ"
    c.check(got, window, sinks)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("many", [4, 60])
def test_long_own_keys_and_a_given_scale(cuda_dev, f8, many):
    """Few sequences whose own keys are long (split over blocks that join in a launch of their own), and many."""
    c = Case(3, cuda_dev, [(64, [70, 9000] + [66] * many)], 4, 1, 64, 16, torch.bfloat16, f8)
    got = ops.prefix_attention(*c.args(), scale=0.3, **c.scales())
    c.check(got, scale=0.3)
    few = Case(4, cuda_dev, [(64, [30000]), (10, [20000])], 4, 1, 64, 16, torch.bfloat16, f8)
    few.check(ops.prefix_attention(*few.args(), **few.scales()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sequences", [3, 70])
def test_what_a_sequence_does_not_see_does_not_reach_it(cuda_dev, dtype, sequences):
    """NaN and infinities in keys and values of the prefix that the window leaves to some sequences of the group only."""
    window, lens = 300, [410 + (17 * i) % 150 for i in range(sequences)]
    c = Case(5, cuda_dev, [(400, lens)], 4, 2, 64, 16, dtype)
    clean = ops.prefix_attention(*c.args(), window=window, sinks=2)
    c.check(clean, window, 2)
    for key in (150, 200, 399, 1):  # 1: a first token, seen by all
        page, offset = c.place(0, key)
        for t, value in ((c.k, math.nan), (c.v, math.inf)):
            keep = t[page, :, offset].clone()
            t[page, :, offset] = value
            got = ops.prefix_attention(*c.args(), window=window, sinks=2)
            sees = torch.tensor([key > n - 1 - window or key < 2 for n in lens])
            assert torch.equal(got.cpu()[~sees], clean.cpu()[~sees]), key
            reached = ~got.cpu()[sees].isfinite().flatten(1)
            assert bool(reached.all(1).all() if value != value else reached.any(1).all()), key
            t[page, :, offset] = keep


@pytest.mark.parametrize("sequences", [3, 70])
def test_extremes(cuda_dev, sequences):
    """Logits of minus infinity give zeros, large ones the value of the largest, and a query of NaN is NaN for its sequence alone."""
    lens = [200 + i for i in range(sequences)]
    c = Case(6, cuda_dev, [(200, [n + 1 for n in lens])], 4, 2, 64, 16, torch.bfloat16)
    clean = ops.prefix_attention(*c.args())
    c.q[1] = math.nan
    got = ops.prefix_attention(*c.args())
    assert bool(got[1].isnan().all()) and torch.equal(got[0].cpu(), clean[0].cpu()) and torch.equal(got[2:].cpu(), clean[2:].cpu())
    c.q[1] = c.q[0]
    c.k[c.k.isnan()] = 0.0
    c.k[:], c.q[:] = 0.0, 0.0
    c.q[..., 0], c.k[..., 0] = 3e38, -3e38  # every product is minus infinity
    assert int(ops.prefix_attention(*c.args()).count_nonzero()) == 0
    for size in (1e3, 1e15):
        d = Case(7, cuda_dev, [(200, [n + 1 for n in lens])], 4, 2, 64, 16, torch.bfloat16)
        d.q[:], d.k[~d.k.isnan()] = d.q.sign() * size, d.k[~d.k.isnan()] * size
        got = ops.prefix_attention(*d.args()).cpu()
        assert not got.isnan().any() and float(got.abs().max()) < 8


def test_the_same_as_attention_over_pages(cuda_dev):
    """With whole pages shared, the tables of paged_attention say the same; and a group for each sequence, or no prefix at all, is paged_attention."""
    g = torch.Generator().manual_seed(8)
    page, hkv, dim, own = 16, 2, 128, [3, 40, 16, 1]
    pages, per = 30, 7
    k, v = (torch.randn(pages, hkv, page, dim, generator=g).bfloat16().to(cuda_dev) for _ in range(2))
    q = torch.randn(4, 8, dim, generator=g).bfloat16().to(cuda_dev)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    prefix, rest = order[:4], order[4 : 4 + 12].view(4, 3)
    table = torch.cat([prefix.expand(4, 4), rest], 1).contiguous().to(cuda_dev)
    lens = torch.tensor([64 + n for n in own], dtype=torch.int32, device=cuda_dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    want = ops.paged_attention(q, k, v, table, lens).float()
    size = 3 * 2.0**-8 * float(v.float().abs().max())  # two ways of one row: weights in 16 bits and one rounding each
    for got in (ops.prefix_attention(q, k, v, prefix.view(1, 4).to(cuda_dev), i32(64), i32(0, 4), table, lens),
                ops.prefix_attention(q, k, v, prefix.expand(4, 4).to(cuda_dev), i32(64, 50, 0, 17), i32(0, 1, 2, 3, 4), table, lens),
                ops.prefix_attention(q, k, v, prefix.view(1, 4).to(cuda_dev)[:, :0], i32(0), i32(0, 4), table, lens)):  # fmt: skip
        assert float((got.float() - want).abs().max()) <= size
    assert per == table.shape[1]


def test_other_layouts_and_outputs(cuda_dev):
    c = Case(9, cuda_dev, [(100, [101, 140]), (30, [31])], 8, 2, 64, 16, torch.bfloat16)
    q, k, v, *rest = c.args()
    want = ops.prefix_attention(q, k, v, *rest)
    k2, v2 = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    assert torch.equal(ops.prefix_attention(q, k2, v2, *rest), want)
    wide = torch.zeros(3, 8, 128, dtype=q.dtype, device=cuda_dev)
    wide[..., :64] = q
    out = torch.empty_like(want)
    assert ops.prefix_attention(wide[..., :64], k, v, *rest, out=out) is out or torch.equal(out, want)
    assert torch.equal(out, want)
    q2 = q.clone()
    assert torch.equal(ops.prefix_attention(q2, k, v, *rest, out=q2), want) and torch.equal(q2, want)
    table = torch.cat([rest[0], rest[0]], 1)[:, : rest[0].shape[1]]  # rows with a pitch
    assert torch.equal(ops.prefix_attention(q, k, v, table, *rest[1:]), want)
    empty = ops.prefix_attention(q[:0], k, v, rest[0][:0], rest[1][:0], rest[2][:1], rest[3][:0], rest[4][:0])
    assert empty.shape == (0, 8, 64)


def test_bad_values_are_reported(cuda_dev):
    c = Case(10, cuda_dev, [(100, [101, 140]), (30, [31])], 8, 2, 64, 16, torch.bfloat16)
    c.k[c.k.isnan()], c.v[c.v.isnan()] = 0.0, 0.0
    good = c.args()
    ops.prefix_attention(*good)
    ops.check_status(cuda_dev)
    for at, values in ((5, ([0, 2, 4], [1, 2, 3], [0, 3, 2], [0, -1, 3], [0, -(1 << 31), 3], [0, 1 << 30, 3], [2, 0, 3])), (4, ([100, -1], [113, 30], [1 << 30, 30])),
                       (7, ([101, -2, 31], [101, 140, 1 << 30]))):  # fmt: skip
        for value in values:
            args = list(good)
            args[at] = torch.tensor(value, dtype=torch.int32, device=cuda_dev)
            ops.prefix_attention(*args)
            with pytest.raises(RuntimeError, match="status"):
                ops.check_status(cuda_dev)
    for at, place in ((3, (0, 2)), (6, (1, 7))):  # a page that does not exist
        for bad in (-1, 1 << 30, c.k.shape[0]):
            args = [t.clone() for t in good]
            args[at][place] = bad
            ops.prefix_attention(*args)
            with pytest.raises(RuntimeError, match="status"):
                ops.check_status(cuda_dev)


def test_bad_values_without_pages_of_a_prefix_are_reported(cuda_dev):
    """No launch for prefixes: the other one looks at the groups and lengths."""
    c = Case(10, cuda_dev, [(0, [20, 40]), (0, [31])], 8, 2, 64, 16, torch.bfloat16)
    good = c.args()
    good[3] = good[3][:, :0]
    c.check(ops.prefix_attention(*good))
    ops.check_status(cuda_dev)
    for at, value in ((4, [0, 5]), (4, [-1, 0]), (5, [0, 1, 2]), (5, [0, 3, 2]), (5, [1, 2, 3])):
        args = list(good)
        args[at] = torch.tensor(value, dtype=torch.int32, device=cuda_dev)
        ops.prefix_attention(*args)
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status(cuda_dev)


def test_refusals(cuda_dev):
    c = Case(11, cuda_dev, [(100, [101, 140]), (30, [31])], 8, 2, 64, 16, torch.bfloat16)
    good = c.args()
    for at, bad in ((0, good[0].float()), (0, good[0].cpu()), (0, good[0][:2]), (1, good[1].half()), (3, good[3].long()), (3, good[3][0]), (4, good[4][:1]), (4, good[4].long()),
                    (5, good[5][:2]), (5, good[5].long()), (6, good[6][:2]), (7, good[7][:2]), (2, good[2][:-1])):  # fmt: skip
        args = list(good)
        args[at] = bad
        with pytest.raises(RuntimeError):
            ops.prefix_attention(*args)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.prefix_attention(good[0].clone().requires_grad_(True), *good[1:])
    with pytest.raises(RuntimeError):
        ops.prefix_attention(*good, scale=-1.0)
    with pytest.raises(RuntimeError):
        ops.prefix_attention(*good, k_scale=torch.ones(2, device=cuda_dev), v_scale=torch.ones(2, device=cuda_dev))


@pytest.mark.parametrize("sequences", [3, 70])
def test_streams_graphs_and_other_lengths(cuda_dev, sequences):
    """A captured call replayed with other lengths, prefixes and queries, while other work goes on, and two graphs that run one after the other."""
    a = Case(12, cuda_dev, [(200, [201 + i for i in range(sequences)])], 8, 2, 128, 16, torch.bfloat16)
    b = Case(13, cuda_dev, [(150, [190 - i % 30 for i in range(sequences)])], 8, 2, 128, 16, torch.bfloat16)
    side = torch.cuda.Stream()
    args = a.args()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.check(ops.prefix_attention(*args))
    torch.cuda.synchronize()
    pages = max(a.k.shape[0], b.k.shape[0])
    held = [torch.zeros((pages, *t.shape[1:]), dtype=t.dtype, device=cuda_dev) if i in (1, 2) else
            torch.zeros((t.shape[0], max(t.shape[1], b.args()[i].shape[1])), dtype=t.dtype, device=cuda_dev) if i in (3, 6) else t.clone() for i, t in enumerate(args)]  # fmt: skip
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(ops.prefix_attention(*held))
    for case in (a, b, a):
        for to, t in zip(held, case.args()):
            to[: t.shape[0], : t.shape[1]].copy_(t) if t.dim() > 1 else to.copy_(t)
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            case.check(out)


def test_offsets_beyond_32_bits(cuda_dev):
    """A cache of more than 2^32 elements; prefix and own pages at both ends of it."""
    dim, page, hkv = 128, 64, 8
    pages = (1 << 32) // (hkv * page * dim) + 40
    g = torch.Generator().manual_seed(14)
    k, v = (torch.zeros(pages, hkv, page, dim, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    at = torch.tensor([pages - 1, 3, pages - 7, 0, pages - 2], dtype=torch.int32)
    small = [torch.randn(5, hkv, page, dim, generator=g).bfloat16().to(cuda_dev) for _ in range(2)]
    for big, s in zip((k, v), small):
        big[at.long().to(cuda_dev)] = s
    q = torch.randn(2, 32, dim, generator=g).bfloat16().to(cuda_dev)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(cuda_dev)  # noqa: E731
    both = [ops.prefix_attention(q, kk, vv, i32([[t[0], t[1]]]), i32([128]), i32([0, 2]), i32([[0, 0, t[2], t[3]], [0, 0, t[4], 0]]), i32([250, 140]))
            for kk, vv, t in ((k, v, at.tolist()), (*small, [0, 1, 2, 3, 4]))]  # fmt: skip
    ops.check_status(cuda_dev)
    assert torch.equal(*both)


@pytest.mark.parametrize("dim,f8", [(8, False), (40, False), (80, False), (112, False), (16, True), (48, True), (80, True), (112, True)])
@pytest.mark.parametrize("sequences", [20, 50])
def test_head_dimensions(cuda_dev, dim, f8, sequences):
    """Head dimensions that fill no tile, with as many rows as one tile of 128 has, and two; what lies between the heads in memory is NaN."""
    c = Case(15, cuda_dev, [(333, [340 + (7 * i) % 60 for i in range(sequences)])], 4, 1, dim, 16, torch.bfloat16, f8)
    args = c.args()
    for i in (1, 2):
        wide = torch.full((*args[i].shape[:3], dim + 16), math.nan, device=cuda_dev).to(args[i].dtype)
        wide[..., :dim] = args[i]
        args[i] = wide[..., :dim]
    c.check(ops.prefix_attention(*args, **c.scales()))
    ops.check_status(cuda_dev)


def test_many_groups(cuda_dev):
    """More groups than a warp looks at in one go, some without sequences, and sequences of no prefix among them."""
    groups = [((i * 13) % 50, [(i * 13) % 50 + 1 + (i + j) % 9 for j in range(i % 4)]) for i in range(150)]
    c = Case(16, cuda_dev, groups, 4, 2, 64, 16, torch.bfloat16)
    c.check(ops.prefix_attention(*c.args()))
    ops.check_status(cuda_dev)
    big = [(300, [310 + i for i in range(33)])] + [(20, [25])] * 40 + [(200, [201 + i for i in range(40)])]
    c = Case(17, cuda_dev, big, 8, 1, 64, 16, torch.float16)
    c.check(ops.prefix_attention(*c.args()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sequences", [3, 20, 70])
@pytest.mark.parametrize("at", [100, 705])
def test_an_infinite_value_of_small_weight(cuda_dev, dtype, sequences, at):
    """A value of infinity that is seen with a weight of 2^-58, too small for fp16, in the prefix or among a sequence's own keys: the output is infinite, not 0 * infinity."""
    c = Case(18, cuda_dev, [(700, [720] * sequences)], 4, 1, 64, 16, dtype)
    c.q[:], c.k[~c.k.isnan()] = 0.0, 0.0
    c.q[..., 0] = 8
    page, offset = c.place(0, at)
    c.k[page, 0, offset, 0] = -40
    c.v[page, 0, offset, 3] = math.inf
    got = ops.prefix_attention(*c.args()).cpu()
    sees = torch.arange(sequences) >= (0 if at < 700 else sequences)
    sees[0] = True
    assert bool((got[sees][..., 3] == math.inf).all()) and bool(got[~sees].isfinite().all())
    assert bool(got[..., [d for d in range(64) if d != 3]].isfinite().all())


@pytest.mark.parametrize("dtype,f8", [(torch.bfloat16, False), (torch.float16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("sequences", [3, 70])
def test_large_logits_a_few_units_apart(cuda_dev, dtype, f8, sequences):
    """Logits whose last place is worth more than the weights' reference may lag behind: every other 128 keys lie 8 above the rest.  Products, sums and differences of logits are exact, so
    the weights are as near as any (2^-20 for their exponents), whatever the logits' size."""
    n, dim = 1024, 64
    c = Case(19, cuda_dev, [(n, [n + 10] * sequences)], 16, 1, dim, 64, dtype, f8)
    high = (torch.arange(n + 10) // 128 % 2 == 1) & (torch.arange(n + 10) < n)
    common, step, q = (256.0, 2.0, (32768.0, 32768.0, 1.0)) if f8 else (16384.0, 8.0, (32768.0, 0.0, 8.0))
    k = torch.zeros(c.k.shape)
    for b in range(sequences):
        for j in range(n if b else 0, n + 10):
            page, offset = c.place(b, j)
            k[page, 0, offset, :2], k[page, 0, offset, 2] = common, step * float(high[j])
    c.k = k.to(c.k.dtype)
    c.q[:] = 0.0
    c.q[..., :3] = torch.tensor(q)
    if f8:
        c.ks[:] = 32.0
    got = ops.prefix_attention(*c.args(), **c.scales()).cpu().double()
    p = torch.softmax(torch.where(high, 8.0, 0.0).double(), 0)
    wt = torch.float16 if f8 else dtype
    for b in range(sequences):
        at = [c.place(b, j) for j in range(n + 10)]
        v = torch.stack([c.v[page, 0, offset].double() for page, offset in at]) * (c.vs[0].double() if f8 else 1.0)
        want, weighted = p @ v, p @ v.abs()
        tol = (2 * U[wt] + 2.0**-20) * weighted + U[dtype] * want.abs() + (n + 10) * 2.0**-30 * v.abs().max() + 2.0**-25
        assert bool(((got[b] - want).abs() <= tol).all()), (b, got[b].isfinite().all(), float((got[b] - want).abs().max()))


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sequences", [8, 48, 136])
def test_many_keys_of_no_weight(cuda_dev, dtype, f8, sequences):
    """A key with all of the weight and a value of zero, and 2^17 with 2^-58 of it and values of one: no output comes of these.  An fp16 weight that is kept from zero, so that an
    infinite value stays one, adds 2^-36 of the largest at most."""
    heads, dim, page, n = 80, 16 if f8 else 8, 64, 1 << 17
    k, v = (torch.zeros(n // page + 1, heads, page, dim, device=cuda_dev) for _ in range(2))
    k[..., 0], v[:] = -8.0, 1.0
    k[0, :, 0, 0], v[0, :, 0] = 0.0, 0.0
    q = torch.zeros(sequences, heads, dim, dtype=dtype, device=cuda_dev)
    q[..., 0] = 58 / 8 * math.log(2) / dim**-0.5
    ct = F8 if f8 else dtype
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    table = torch.arange(n // page, dtype=torch.int32, device=cuda_dev)
    own = torch.zeros(sequences, n // page + 1, dtype=torch.int32, device=cuda_dev)
    own[:, -1] = n // page
    scales = dict(k_scale=torch.ones(heads, device=cuda_dev), v_scale=torch.ones(heads, device=cuda_dev)) if f8 else {}
    got = ops.prefix_attention(q, k.to(ct), v.to(ct), table[None], i32(n), i32(0, sequences), own, i32(*[n + 3] * sequences), **scales)
    ops.check_status(cuda_dev)
    assert float(got.abs().max()) <= (n + 3) * 2.0**-36 + 2.0**-25
