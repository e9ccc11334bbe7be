"""How the kernels of experts share a line of stages, and which kernel takes an int8 product: csrc/experts_parts.cuh and csrc/qlinear_i8_plan.h, run on the host."""
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope='module')
def ask(tmp_path_factory):
    out = str(tmp_path_factory.mktemp('parts') / 'parts')
    subprocess.check_call([os.environ.get('CXX', 'g++'), '-O1', '-std=c++17', os.path.join(HERE, 'host', 'experts_parts.cpp'), '-o', out])

    def run(lines):
        answer = subprocess.run([out], input='\n'.join(' '.join(map(str, line)) for line in lines), stdout=subprocess.PIPE, text=True, timeout=120, check=True).stdout
        return [list(map(int, line.split())) for line in answer.splitlines()]

    return run


def check_line(entries, tiles, k_blocks, ctas, down, total, step, numbers):
    """Every stage has one CTA, parts are equal up to a piece, and of what CTAs share each holds its part in a place of its own, where the others look for it."""
    first, owner = numbers[:ctas + 1], numbers[ctas + 1:]
    assert first[0] == 0 and first[-1] == total == entries * tiles * k_blocks
    sizes = [b - a for a, b in zip(first, first[1:])]
    assert min(sizes) >= 0 and max(sizes) - min(sizes) <= step
    if step > 1:  # whole units: hardly more than an equal part
        assert not down and step == k_blocks and max(sizes) <= total // ctas + 10 and all(f % k_blocks == 0 for f in first)
        return
    if owner:
        assert owner == [c for c in range(ctas) for _ in range(sizes[c])]
    shared = k_blocks * (entries if down else 1)  # stages of what is brought together: a unit, or a column tile's units
    places, holders = {}, {}
    for c in range(ctas):
        if sizes[c] == 0:
            continue
        for u in range(first[c] // shared, (first[c + 1] - 1) // shared + 1):
            if first[c] <= u * shared and (u + 1) * shared <= first[c + 1]:
                continue  # this CTA's alone
            place = (c, first[c] < u * shared)
            assert place not in places
            places[place] = u
            holders.setdefault(u, []).append(c)
    for u, own in holders.items():
        # what a CTA that shares u computes of who else does
        a, b = (next(c for c in range(ctas) if first[c] <= s < first[c + 1]) for s in (u * shared, (u + 1) * shared - 1))
        assert own == list(range(a, b + 1))
    firsts = [min(own) for own in holders.values()]
    assert len(firsts) == len(set(firsts))  # arrivals are counted by the first of them


def test_parts_of_a_line(ask):
    rng = random.Random(3)
    cases = [(2, 224, 32, 148, 0), (2, 32, 112, 148, 1), (122, 12, 16, 148, 0), (122, 16, 6, 148, 1), (1, 1, 1, 148, 0), (1, 1, 1, 148, 1), (6, 22, 16, 148, 0), (0, 5, 3, 148, 1), (1, 2, 200, 148, 1)]
    cases += [(rng.randint(1, 12), rng.randint(1, 12), rng.randint(1, 9), rng.choice([1, 2, 5, 13, 37, 148]), rng.randint(0, 1)) for _ in range(1500)]
    for (entries, tiles, k_blocks, ctas, down), numbers in zip(cases, ask([('parts', e * t, k, c, int(not d)) for e, t, k, c, d in cases])):
        if entries:
            check_line(entries, tiles, k_blocks, ctas, down, numbers[0], numbers[1], numbers[2:])
        else:
            assert not any(numbers[2:])


@pytest.mark.parametrize('sms', [148, 132, 20])
def test_plan_of_a_product(ask, sms):
    """Every size has a form that its kernel takes: tile sizes in their steps, shares of K that are not empty, and pairs that share K with a place each."""
    rng = random.Random(sms)
    sizes = [(m, n, k) for m in (1, 16, 17, 64, 65, 256, 1000, 8192) for n in (16, 4096, 28672) for k in (16, 4096, 131056)]
    sizes += [(int(10 ** rng.uniform(0, 5)), 16 * int(10 ** rng.uniform(0, 3.3)), 16 * int(10 ** rng.uniform(0, 3.9))) for _ in range(3000)]
    seen = set()
    for (m, n, k), (pair, tm, split) in zip(sizes, ask([('plan', m, n, k, sms) for m, n, k in sizes])):
        seen.add((pair, split))
        assert 0 < tm <= 256 and 1 <= split <= -(-k // 128)
        if pair:
            assert tm % 32 == 0 and split in (1, 2, 4)
            assert split == 1 or -(-n // 256) * -(-m // tm) * split * 2 <= sms
        else:
            assert tm % 16 == 0 and split in (1, 2, 4, 8)
    if sms == 148:  # where the forms were timed, none is without a size
        assert seen == {(p, s) for p, most in ((0, 8), (1, 4)) for s in (1, 2, 4, 8) if s <= most}


def test_rounds_of_units(ask):
    """Every unit's k has every block once, in parts that are not empty, by pairs whose number in a row says who shares it; a pair's units ascend, and the shared one is its last."""
    rng = random.Random(4)
    cases = [(896, 32, 74, 16), (128, 112, 74, 16), (256, 112, 74, 64), (64, 4, 74, 64), (8, 16, 74, 64), (1, 1, 74, 16), (0, 7, 74, 16), (1, 1024, 74, 80), (74, 3, 74, 80), (75, 200, 74, 16)]
    cases += [(rng.randint(0, 400), rng.randint(1, 130), rng.choice([1, 3, 10, 66, 74]), 16 * rng.randint(1, 5)) for _ in range(1500)]
    shared_somewhere = False
    for (units, k_blocks, pairs, slots), numbers in zip(cases, ask([('rounds',) + c for c in cases])):
        parts, at = {}, 1
        for pair in range(pairs):
            count, mine = numbers[at], numbers[at + 1:at + 1 + 4 * numbers[at]]
            at += 1 + 4 * count
            own = [mine[i:i + 4] for i in range(0, len(mine), 4)]
            assert all(a[0] < b[0] for a, b in zip(own, own[1:])) and all(split == 1 for _, _, _, split in own[:-1])
            for unit, first, last, split in own:
                assert 0 <= first < last <= k_blocks
                parts.setdefault(unit, []).append((first, last, pair, split))
        assert at == len(numbers) and sorted(parts) == list(range(units))
        for unit, own in parts.items():
            split = own[0][3]
            shared_somewhere |= split > 1
            assert len(own) == split and all(s == split for _, _, _, s in own) and own[0][0] == 0 and own[-1][1] == k_blocks
            assert all(a[1] == b[0] for a, b in zip(own, own[1:]))
            first = own[0][2]
            assert split == 1 or (first % split == 0 and [pair for _, _, pair, _ in own] == list(range(first, first + split)))
    assert shared_somewhere


def test_entries_of_an_expert(ask):
    counts = list(range(1, 8193))
    for count, numbers in zip(counts, ask([('entries', c, 0, 0, 0) for c in counts])):
        slots, size, sizes, rooms = numbers[0], numbers[1], numbers[2::2], numbers[3::2]
        assert sum(sizes) == count and sum(rooms) == slots and len(sizes) == -(-count // 80)
        assert all(s == size for s in sizes[:-1]) and 1 <= sizes[-1] <= size <= 80 and all(r == -(-s // 16) * 16 for s, r in zip(sizes, rooms))
