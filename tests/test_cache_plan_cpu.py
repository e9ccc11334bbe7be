"""The plan of attention over the quantized cache (csrc/cache_plan.cuh), run on the host: who takes which tiles, whatever a call has on the device."""
import os
import random
import subprocess
from collections import defaultdict, namedtuple

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
TILE = 64
Piece = namedtuple('Piece', 'cta sequence head row0 rows token0 length fresh first_cta last_cta slot tile0 tiles')


@pytest.fixture(scope='module')
def program(tmp_path_factory):
    out = str(tmp_path_factory.mktemp('plan') / 'cache_plan')
    subprocess.check_call([os.environ.get('CXX', 'g++'), '-O1', '-std=c++17', os.path.join(HERE, 'host', 'cache_plan.cpp'), '-o', out])
    return out


def plan(program, rows, grid, lengths, tokens, starts=None, kv_heads=2, group=4, capacity=1 << 17):
    """(pieces, status word)."""
    batch = len(lengths)
    numbers = [rows, grid, batch, kv_heads, group, tokens, capacity, tokens // batch if starts is None else 0, int(starts is not None)] + (starts or []) + lengths
    out = subprocess.run([program], input=' '.join(map(str, numbers)), stdout=subprocess.PIPE, text=True, timeout=120, check=True).stdout.splitlines()
    return [Piece(*map(int, line.split())) for line in out[:-1]], int(out[-1].split()[1])


def most_tiles(rows, lengths, tokens, kv_heads, group, capacity):
    return kv_heads * (tokens * group // rows + len(lengths)) * (capacity // TILE + 1)


def check(pieces, rows, lengths, starts, kv_heads, group):
    """Every tile of every item once, the pieces of an item in CTAs that follow one another, and a place of its own for each."""
    items = defaultdict(list)
    for p in pieces:
        items[p.sequence, p.head, p.row0].append(p)
    want = {(b, h, r) for b in range(len(lengths)) for h in range(kv_heads) for r in range(0, (starts[b + 1] - starts[b]) * group, rows)}
    assert set(items) == want
    places = set()
    for (b, _, row0), own in items.items():
        fresh = starts[b + 1] - starts[b]
        at = 0
        for i, p in enumerate(own):
            assert p.tile0 == at and p.tiles > 0
            at += p.tiles
            assert (p.rows, p.token0, p.length, p.fresh) == (min(rows, fresh * group - row0), starts[b], max(0, lengths[b]), fresh)
            assert p.cta == own[0].cta + i and (p.first_cta, p.last_cta) == (own[0].cta, own[-1].cta)
            if len(own) > 1:
                assert p.slot == 2 * p.cta + (i == 0) and p.slot not in places
                places.add(p.slot)
        assert at == max(1, -(-lengths[b] // TILE))


@pytest.mark.parametrize('rows,grid', [(8, 444), (16, 296), (128, 148)])
@pytest.mark.parametrize('lengths,fresh', [([1], [1]), ([577], [1]), ([131071], [3]), ([0, 0], [1, 0]), ([90, 4000, 16, 0, 333, 64, 65], [1, 3, 0, 2, 60, 1, 1]),
                                           ([700] * 70, [1] * 70), ([64 * (i % 9) for i in range(1000)], [i % 3 for i in range(1000)]), ([4096] * 8, [64] * 8), ([5000, 3], [2000, 2])])
def test_every_tile_is_taken_once(program, rows, grid, lengths, fresh):
    starts = [sum(fresh[:b]) for b in range(len(fresh) + 1)]
    for kv_heads, group, front, behind in ((1, 1, 0, 0), (8, 4, 2, 5)):
        tokens = starts[-1] + front + behind
        at = [s + front for s in starts]
        ctas = min(grid, most_tiles(rows, lengths, tokens, kv_heads, group, 1 << 17))
        pieces, status = plan(program, rows, ctas, lengths, tokens, at, kv_heads, group)
        check(pieces, rows, lengths, at, kv_heads, group)
        assert status == 0
        if len(set(fresh)) == 1 and not front:
            assert plan(program, rows, ctas, lengths, tokens, None, kv_heads, group) == (pieces, 0)


def test_random_batches(program):
    rng = random.Random(5)
    for _ in range(40):
        rows, grid = rng.choice([(8, 444), (16, 296), (128, 148), (8, 3), (128, 2)])
        batch = rng.choice([1, 2, 31, 32, 33, 64, 100])
        lengths = [int(2 ** rng.uniform(0, 14)) for _ in range(batch)]
        fresh = [rng.choice([0, 1, 1, 1, 7, 40]) for _ in range(batch)]
        starts = [sum(fresh[:b]) for b in range(batch + 1)]
        kv_heads, group = rng.choice([1, 2, 8]), rng.choice([1, 4, 5])
        pieces, status = plan(program, rows, grid, lengths, max(1, starts[-1]), starts, kv_heads, group)
        check(pieces, rows, lengths, starts, kv_heads, group)
        assert status == 0


def test_lengths_beyond_the_page_table(program):
    pieces, status = plan(program, 8, 5, [10 ** 9, -3, 100], 3, None, 1, 1, capacity=640)
    check(pieces, 8, [640, -3, 100], [0, 1, 2, 3], 1, 1)
    assert status == 1 << 27


@pytest.mark.parametrize('rows,grid', [(8, 444), (16, 296), (128, 148)])
@pytest.mark.parametrize('starts', [[0, 4096] * 32 + [0], [4096] * 64 + [0], [0] * 64 + [4097], [-1] + [4096] * 64, [0, 5] + [3] * 62 + [9], [2 ** 31 - 1] * 65, [-2 ** 31] * 65,
                                    [0] * 40 + [4096, 4095] + [4096] * 23, list(range(4096, 4096 - 65, -1))], ids=lambda s: '{}_{}_{}'.format(s[0], s[1], s[-1]))
def test_starts_out_of_order_or_range(program, rows, grid, starts):
    """Nothing is planned, and the status word tells.  (The first of these claims every row 32 times over, more tiles than 32 bits count.)"""
    pieces, status = plan(program, rows, grid, [131072] * 64, 4096, starts, 8, 8)
    assert not pieces and status == 1 << 25


@pytest.mark.parametrize('rows,grid', [(8, 444), (128, 148)])
def test_rows_without_a_sequence(program, rows, grid):
    for starts in ([0, 0, 0], [9, 9, 9]):
        assert plan(program, rows, grid, [100, 200], 9, starts) == ([], 0)


def test_random_starts(program):
    rng = random.Random(9)
    for _ in range(60):
        rows, grid = rng.choice([(8, 20), (128, 9)])
        batch = rng.choice([1, 2, 33, 64])
        starts = sorted(rng.randint(0, 50) for _ in range(batch + 1))
        if rng.random() < 0.5:
            starts[rng.randrange(batch + 1)] = rng.choice([-5, 7, 60])
        lengths = [rng.randint(0, 500) for _ in range(batch)]
        fine = starts == sorted(starts) and 0 <= starts[0] and starts[-1] <= 50
        pieces, status = plan(program, rows, grid, lengths, 50, starts, 2, 3)
        assert status == (0 if fine else 1 << 25)
        if fine:
            check(pieces, rows, lengths, starts, 2, 3)
        else:
            assert not pieces
