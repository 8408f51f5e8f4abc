"""Requests of the paged cache that go on from others, by the rule; the copies of begun blocks."""

import random

import pytest
import torch

import kv8_plain as P
import ojasx_amd
import reorder_plain as R
from ojasx_amd import kv8, serve_ops as S

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _check(parents, lens, tables, free, num_free, block, blocks):
    width = tables.shape[1] if isinstance(tables, torch.Tensor) else len(tables[0])
    t = tables if isinstance(tables, torch.Tensor) else _i32(tables).reshape(len(lens), width)
    par = torch.tensor(parents, dtype=torch.int64, device=DEV)
    got = kv8.reorder(par, _i32(lens), t, _i32(free), _i32([num_free]), block, blocks)
    want = R.reorder(parents, lens, t.tolist() if len(lens) else [], free, num_free, block, blocks)
    if not len(lens):
        want = ([[-1] * width for _ in parents], *want[1:])
    assert got.block_tables.shape == (len(parents), width)
    assert got.block_tables.tolist() == want[0]
    assert got.seq_lens.tolist() == want[1]
    assert got.num_free.tolist() == [want[3]]
    assert got.free_blocks.tolist() == want[2]
    assert got.sources.tolist() == want[4]
    assert got.targets.tolist() == want[5]
    op = S.kv8_reorder(par, _i32(lens), t, _i32(free), _i32([num_free]), block, blocks)
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, op))
    return got


def _batch(rng, rows, width, block, blocks, share=0.5, most=None):
    """Rows that share full blocks, their begun blocks their own; the rest on the stack."""
    pool = list(range(blocks))
    rng.shuffle(pool)
    lens, tables = [], []
    for r in range(rows):
        n = rng.randint(0, min(most or width * block, width * block))
        used, full = -(-n // block), n // block
        row = []
        if r and rng.random() < share:
            other = rng.randrange(r)
            row = tables[other][:min(full, lens[other] // block)]
        if used - len(row) > len(pool):
            n, row, used = 0, [], 0
        row = row + [pool.pop() for _ in range(used - len(row))]
        tables.append(row + [rng.choice([-1, 5, 10 ** 9]) for _ in range(width - len(row))])
        lens.append(n)
    return lens, tables, pool


@pytest.mark.parametrize("rows,children,width,block,blocks", [
    (1, 1, 1, 16, 1), (1, 4, 6, 16, 40), (4, 4, 5, 32, 60), (16, 16, 34, 64, 700), (16, 3, 9, 16, 200),
    (3, 40, 9, 256, 33), (64, 64, 200, 16, 9000), (300, 257, 20, 32, 3000), (1500, 2100, 7, 16, 9000),
    (5, 5, 3000, 16, 14000), (40, 40, 30, 16, 500001)])
def test_rows_that_go_on(rows, children, width, block, blocks):
    rng = random.Random(rows * 1000 + width)
    for most in (None, width * block // 3 or 1, 2 * block):
        lens, tables, pool = _batch(rng, rows, width, block, blocks, most=most)
        for parents in ([rng.randrange(rows) for _ in range(children)],
                        [min(rng.randrange(rows), rng.randrange(rows)) if rng.random() < 0.8 else -1
                         for _ in range(children)],
                        [rng.choice([-1, rows, -5, 10 ** 12, rows - 1]) for _ in range(children)],
                        [i if i < rows else -1 for i in range(children)]):
            _check(parents, lens, tables, pool, len(pool), block, blocks)


def test_stacks_that_are_short():
    rng = random.Random(5)
    for trial in range(20):
        lens, tables, pool = _batch(rng, 6, 4, 16, 30)
        parents = [rng.randrange(6) for _ in range(9)]
        for n in (len(pool), 3, 1, 0, -2):
            _check(parents, lens, tables, pool, n, 16, 30)
        _check(parents, lens, tables, pool[:2], 5, 16, 30)
        _check(parents, lens, tables, [], 0, 16, 30)
    # one prompt for four beams, with a block for one of them only
    got = _check([0, 0, 0, 0], [20], [[3, 4]], [7], 1, 16, 8)
    assert got.targets.tolist() == [-1, 7, -1, -1] and got.num_free.tolist() == [-2]
    assert got.block_tables.tolist() == [[3, 4], [3, 7], [3, -1], [3, -1]]


def test_rows_out_of_the_ordinary():
    # no rows, no children, tables without columns, longer requests than tables hold, lengths below 0
    _check([], [20, 5], [[3, 4], [5, 6]], [7], 1, 16, 8)
    _check([0, -1, 2], [], torch.zeros(0, 4, dtype=torch.int32, device=DEV), [7, 1], 2, 16, 8)
    _check([0, 0], [20], torch.zeros(1, 0, dtype=torch.int32, device=DEV), [7, 1], 2, 16, 8)
    _check([0, 0, 1], [70, -9], [[3, 4], [5, 6]], [7, 1], 2, 16, 8)
    _check([0, 0, 1, 1], [20, 36], [[3, -1], [99, 6]], [7, 1], 2, 16, 8)
    _check([1, 1, 1], [16, 32], [[3, -1], [2, 6]], [7, 1], 2, 16, 8)   # full blocks need no copy
    _check([1, 1, 1], [16, 32], [[3, -1], [2, 6]], [], 0, 16, 0)        # a cache without blocks
    wide = torch.full((4, 12), -7, dtype=torch.int32, device=DEV)
    wide[:, 2:5] = _i32([[0, 1, 2], [0, 1, 3], [0, 4, 5], [6, 7, 8]])
    lens = [40, 41, 48, 33]
    _check([1, 1, 0, 3, 3], lens, wide[:, 2:5], [11, 10, 9], 3, 16, 12)
    _check([1, 1, 0, 3, 3], lens, wide[:, 2:5].t().contiguous().t(), [11, 10, 9], 3, 16, 12)


@pytest.mark.parametrize("heads,d,block,layers", [(1, 64, 16, 1), (2, 80, 16, 3), (4, 128, 64, 2),
                                                  (3, 200, 32, 5), (1, 8, 256, 70)])
def test_copies(heads, d, block, layers):
    blocks = 40
    g = torch.Generator().manual_seed(d)
    caches = [ojasx_amd.KV8Cache(blocks, heads, d, block, DEV) for _ in range(layers)]
    for c in caches:
        P.fill(c, g)
    order = torch.randperm(blocks, generator=g).tolist()
    for n in (0, 1, 5, 19):
        sources = [order[i % 3] if i % 4 else -1 for i in range(n)] + [2, 40, -1, 3]
        targets = [order[3 + i] if i % 5 != 2 else 99 for i in range(n)] + [-1, 1, 4, 40]
        sources += [order[0]] * 100 if n == 19 else []   # more than 64 pairs, most of them nothing
        targets += [-1] * 99 + [order[30]] if n == 19 else []
        want = []
        for c in caches:
            kept = [t.clone() for t in (c.k_codes, c.v_codes, c.scales)]
            for s, t in zip(sources, targets):
                if 0 <= s < blocks and 0 <= t < blocks:
                    for x in kept:
                        x[t] = x[s]
            want.append(kept)
        version = caches[0].k_codes._version
        as_parts = [(c.k_codes, c.v_codes, c.scales) for c in caches]
        kv8.copy_blocks(caches if n % 2 else as_parts, _i32(sources), _i32(targets))
        assert caches[0].k_codes._version > version
        for c, kept in zip(caches, want):
            assert all(torch.equal(a, b) for a, b in zip((c.k_codes, c.v_codes, c.scales), kept))
    # the registered op
    other = [ojasx_amd.KV8Cache(blocks, heads, d, block, DEV) for _ in range(layers)]
    for a, b in zip(other, caches):
        for x, y in ((a.k_codes, b.k_codes), (a.v_codes, b.v_codes), (a.scales, b.scales)):
            x.copy_(y)
    pair = _i32([1, 2, -1]), _i32([3, 4, 5])
    kv8.copy_blocks(caches, *pair)
    S.kv8_copy_blocks([c.k_codes for c in other], [c.v_codes for c in other],
                      [c.scales for c in other], *pair)
    for a, b in zip(other, caches):
        assert torch.equal(a.k_codes, b.k_codes) and torch.equal(a.v_codes, b.v_codes)
        assert torch.equal(a.scales, b.scales)
    kv8.copy_blocks([], *pair)
    kv8.copy_blocks(caches, *(t[:0] for t in pair))


def test_large_blocks_beyond_32_bits():
    """The last of blocks whose codes lie past 2^31 bytes."""
    c = ojasx_amd.KV8Cache(9, 64, 256, 256, DEV)      # 4 MiB a block
    big = ojasx_amd.KV8Cache(600, 64, 256, 256, DEV)  # 2.3 GiB of keys
    P.fill(c, torch.Generator().manual_seed(1))
    for x, y in ((big.k_codes, c.k_codes), (big.v_codes, c.v_codes), (big.scales, c.scales)):
        x[7:9] = y[:2]
    kv8.copy_blocks([big], _i32([7, 8]), _i32([599, 530]))
    for x in (big.k_codes, big.v_codes, big.scales):
        assert torch.equal(x[599], x[7]) and torch.equal(x[530], x[8]) and x[600 - 2].abs().max() == 0


def test_in_a_graph_and_on_a_stream():
    rng = random.Random(8)
    batches = [_batch(rng, 12, 6, 16, 90) for _ in range(5)]
    caches = [ojasx_amd.KV8Cache(90, 2, 64, 16, DEV) for _ in range(3)]
    for c in caches:
        P.fill(c, torch.Generator().manual_seed(2))
    lens, tables, pool = batches[0]
    state = [torch.tensor([rng.randrange(12) for _ in range(16)], device=DEV), _i32(lens), _i32(tables),
             _i32(pool + [0] * (90 - len(pool))), _i32([len(pool)])]

    def step():
        r = kv8.reorder(*state, 16, 90)
        kv8.copy_blocks(caches, r.sources, r.targets)
        return r

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens, tables, pool in batches[1:]:
        for x, y in zip(state, ([rng.randrange(-1, 12) for _ in range(16)], lens, tables,
                                pool + [0] * (90 - len(pool)), [len(pool)])):
            x.copy_(torch.tensor(y, device=DEV))
        before = [c.k_codes.clone() for c in caches]
        graph.replay()
        torch.cuda.synchronize()
        want = kv8.reorder(*state, 16, 90)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        on = want.targets >= 0
        for c, b in zip(caches, before):
            b[want.targets[on].long()] = b[want.sources[on].long()]
            assert torch.equal(c.k_codes, b)


def test_refusals():
    par = torch.zeros(3, dtype=torch.int64, device=DEV)
    good = (par, _i32([20, 3]), _i32([[0, 1], [2, 3]]), _i32([5, 6]), _i32([2]), 16, 8)
    kv8.reorder(*good)
    for i, bad in ((0, par.int()), (0, par[None]), (0, par.cpu()), (1, par), (1, _i32([1])), (1, _i32([[1, 2]])),
                   (2, par[None].expand(2, 3)), (2, _i32([[0, 1]])), (2, _i32([0, 1])), (3, par),
                   (4, _i32([1, 2])), (5, 24), (6, -1)):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError):
            kv8.reorder(*args)
    c, other = ojasx_amd.KV8Cache(4, 2, 64, 16, DEV), ojasx_amd.KV8Cache(5, 2, 64, 16, DEV)
    one = _i32([1])
    for args in (([c], one.long(), one), ([c], one, _i32([1, 2])), ([c], one, one.cpu()),
                 ([c, other], one, one), ([(c.k_codes, c.v_codes)], one, one),
                 ([(c.k_codes, c.v_codes, c.scales[:3])], one, one),
                 ([(c.k_codes, c.v_codes.float(), c.scales)], one, one),
                 ([ojasx_amd.KV8Cache(4, 2, 64, 16, "cpu")], one, one)):
        with pytest.raises(RuntimeError):
            kv8.copy_blocks(*args)
