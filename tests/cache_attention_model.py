"""Host-side models of the two kernels of attention over the quantized cache, in the manner of pipeline_model.py: which barrier each role waits on, with
which parity, what it signals and what it then finds in each buffer, under random schedules in which copies land late and out of order and any wait may run out.

`ManyRows` is cache_attention_wide.cu, `FewRows` cache_attention.cu.  Work is a list of items, each its number of tiles.  Test infrastructure only."""
from __future__ import annotations

import os
import random
import re
from dataclasses import dataclass
from typing import Dict, List, Optional

from pipeline_model import KERNELS, Aborted, Barrier, Meeting, ProtocolError, Scheduler, _constants

GROUPS, WARPS = 2, 4


@dataclass
class ManyRowsConfig:
    raw_stages: int
    kv_stages: int
    items: int
    ahead: int
    agrees: bool = True           # warps that meet at the named barrier bring whether their waits gave up, and leave there
    drains: str = 'always'        # when the warp that copies waits for its copies: 'always', where its 'own' wait ran out, 'never'
    ends_by_item: bool = True     # the end of an item is waited for by a barrier of its own; False: by the last product's


def drains_in_source(name: str) -> str:
    """Whether the loop over the last stages, in which the copying warp waits for its copies, stands under a condition."""
    text = open(os.path.join(KERNELS, name)).read()
    found = re.search(r'( *)(if \([^\n]*\) \{[^\n]*\n)? *for \(int back = 1; ', text)
    return 'never' if found is None else 'own' if found.group(2) else 'always'


def many_rows_config_from_source() -> ManyRowsConfig:
    k = _constants(open(os.path.join(KERNELS, 'cache_attention_wide.cu')).read())
    assert k['GROUP_WARPS'] == WARPS
    return ManyRowsConfig(raw_stages=k['RAW_STAGES'], kv_stages=k['KV_STAGES'], items=k['ITEMS'], ahead=k['AHEAD'], drains=drains_in_source('cache_attention_wide.cu'))


def expect(found, wanted, what: str):
    if found != wanted:
        raise ProtocolError('{}: found {}, not {}'.format(what, found, wanted))


class Kernel(Scheduler):
    """What both have: the warp that copies tiles and tells of items, and the exit."""

    def __init__(self, rng: random.Random, work: List[int], stages: int, items: int, raw_readers: int, item_readers: int):
        super().__init__(rng)
        self.work, self.stages = work, stages
        self.raw_full = [Barrier('raw_full[{}]'.format(s), 1) for s in range(stages)]
        self.raw_empty = [Barrier('raw_empty[{}]'.format(s), raw_readers) for s in range(stages)]
        self.item_full = [Barrier('item_full[{}]'.format(s), 1) for s in range(items)]
        self.item_empty = [Barrier('item_empty[{}]'.format(s), item_readers) for s in range(items)]
        self.raw: List[Optional[int]] = [None] * stages   # the tile in it, -1: no more
        self.told: List[Optional[int]] = [None] * items   # the item in it
        self.agents: List = []

    def roles(self):
        return self.agents

    def item_wait(self, n: int):
        return lambda: self.item_full[n % len(self.told)].test((n // len(self.told)) & 1)

    def read_item(self, n: int) -> Optional[int]:
        """Tiles of item n, None behind the last.  The caller has waited; it frees the place."""
        at = n % len(self.told)
        expect(self.told[at], n, 'item')
        self.item_empty[at].arrive()
        return self.work[n] if n < len(self.work) else None

    def publish(self, n: int):
        at = n % len(self.told)
        if n >= len(self.told):
            yield lambda: self.item_empty[at].test((n // len(self.told) - 1) & 1)
        self.told[at] = n
        yield None
        self.item_full[at].arrive()

    def producer(self, tells_end: bool, drains: str):
        it, own = 0, False
        try:
            for n, tiles in enumerate(self.work):
                yield from self.publish(n)
                for _ in range(tiles):
                    s = it % self.stages
                    if it >= self.stages:
                        yield lambda s=s, p=(it // self.stages - 1) & 1: self.raw_empty[s].test(p)
                    self.raw_full[s].arrive_expect_tx(1)

                    def land(s=s, it=it):
                        self.raw[s] = it
                        self.raw_full[s].complete_tx(1)

                    self.copies.append(land)
                    yield None
                    it += 1
            yield from self.publish(len(self.work))
            if tells_end:
                s = it % self.stages
                if it >= self.stages:
                    yield lambda: self.raw_empty[s].test((it // self.stages - 1) & 1)
                self.raw[s] = -1
                self.raw_full[s].arrive()
        except Aborted:
            own = True
        if drains == 'always' or (drains == 'own' and own):
            last = self.stages - 1 if tells_end and not own else self.stages   # the stage that tells of the end was empty for that
            for at in range(it - 1, max(-1, it - 1 - last), -1):
                yield ('drain', lambda: self.raw_full[at % self.stages].test((at // self.stages) & 1))


class ManyRows(Kernel):
    def __init__(self, cfg: ManyRowsConfig, work: List[int], rng: random.Random):
        super().__init__(rng, work, cfg.raw_stages, cfg.items, WARPS, GROUPS * WARPS + 1)
        self.cfg = cfg
        kv = range(cfg.kv_stages)
        self.kv_full = [Barrier('kv_full[{}]'.format(s), WARPS) for s in kv]
        self.kv_empty = [Barrier('kv_empty[{}]'.format(s), 1) for s in kv]
        self.q_full = Barrier('q_full', GROUPS * WARPS)
        self.s_full = [[Barrier('s_full[{}][{}]'.format(g, b), 1) for b in range(2)] for g in range(GROUPS)]
        self.p_full = [[Barrier('p_full[{}][{}]'.format(g, b), WARPS) for b in range(2)] for g in range(GROUPS)]
        self.pv_done = [Barrier('pv_done[{}]'.format(g), 1) for g in range(GROUPS)]
        self.item_done = Barrier('item_done', 1)
        self.kv: List[Dict[int, int]] = [{} for _ in kv]              # warp -> the tile it wrote there
        self.scores = [[{} for _ in range(2)] for _ in range(GROUPS)]   # warp -> ('S' or 'P', tile): its rows
        self.q: Dict[tuple, int] = {}                                 # (group, warp) -> item
        self.o: List[List[int]] = [[], []]                            # tiles that a group's sums hold
        self.meeting, self.exit = Meeting(GROUPS * WARPS), Meeting(2 + WARPS + GROUPS * WARPS)
        roles = [self.producer(True, cfg.drains), self.products()]
        roles += [self.converter(w) for w in range(WARPS)] + [self.softmax(g, w) for g in range(GROUPS) for w in range(WARPS)]
        self.agents = [self.whole(role) for role in roles]

    def whole(self, role):
        try:
            yield from role
        except Aborted:
            pass
        yield self.exit.come()[1]   # __syncthreads in front of giving tensor memory back

    def converter(self, warp: int):
        c, it = self.cfg, 0
        while True:
            s, buf = it % c.raw_stages, it % c.kv_stages
            yield lambda: self.raw_full[s].test((it // c.raw_stages) & 1)
            if self.raw[s] == -1:
                return
            expect(self.raw[s], it, 'converter, raw tile')
            if it >= c.kv_stages:
                yield lambda: self.kv_empty[buf].test((it // c.kv_stages - 1) & 1)
            self.kv[buf] = dict(self.kv[buf])
            self.kv[buf][warp] = it
            yield None
            expect(self.raw[s], it, 'converter, raw tile at its end')
            self.kv_full[buf].arrive()
            self.raw_empty[s].arrive()
            yield None
            it += 1

    def products(self):
        try:
            yield from self._products()
        except Aborted:
            pass
        if self.cfg.drains != 'never':
            yield ('drain', lambda: not self.commits)

    def _products(self):
        c, n, kv, item = self.cfg, [0, 0], 0, 0
        while True:
            yield self.item_wait(item)
            tiles = self.read_item(item)
            if tiles is None:
                return
            yield lambda: self.q_full.test(item & 1)
            asked = 0
            for i in range(tiles):
                while asked < min(tiles, i + c.ahead + 1):
                    g, tile, at = asked & 1, kv + asked, n[asked & 1] + (asked >> 1)
                    buf = tile % c.kv_stages
                    yield lambda: self.kv_full[buf].test((tile // c.kv_stages) & 1)

                    def scored(g=g, tile=tile, at=at, buf=buf, item=item):
                        expect(self.kv[buf], {w: tile for w in range(WARPS)}, 'first product, K')
                        expect(set(self.q.values()), {item}, 'first product, Q')
                        self.scores[g][at & 1] = {w: ('S', tile) for w in range(WARPS)}
                        self.s_full[g][at & 1].arrive()

                    expect(self.kv[buf], {w: tile for w in range(WARPS)}, 'first product, K as it is issued')
                    self.commits.append(scored)
                    yield None
                    asked += 1
                g, tile, at = i & 1, kv + i, n[i & 1] + (i >> 1)
                buf = tile % c.kv_stages
                yield lambda: self.p_full[g][at & 1].test((at >> 1) & 1)

                def added(g=g, tile=tile, at=at, buf=buf, first=i < 2):
                    expect(self.kv[buf], {w: tile for w in range(WARPS)}, 'second product, V')
                    expect(self.scores[g][at & 1], {w: ('P', tile) for w in range(WARPS)}, 'second product, P')
                    self.o[g] = [tile] if first else self.o[g] + [tile]
                    self.pv_done[g].arrive()
                    self.kv_empty[buf].arrive()

                expect(self.scores[g][at & 1], {w: ('P', tile) for w in range(WARPS)}, 'second product, P as it is issued')
                self.commits.append(added)
                yield None
            self.commits.append(self.item_done.arrive)
            yield None
            kv += tiles
            n[0] += (tiles + 1) >> 1
            n[1] += tiles >> 1
            item += 1

    def meet(self, alive: bool = True):
        """The answer of all warps at the named barrier."""
        number, wait = self.meeting.come(alive)
        yield wait
        return self.meeting.results[number] if self.cfg.agrees else True

    def softmax(self, g: int, warp: int):
        met = [False]
        try:
            yield from self._softmax(g, warp, met)
        except Aborted:
            if self.cfg.agrees and not met[0]:
                yield from self.meet(False)

    def _softmax(self, g: int, warp: int, met):
        c, n, kv, item = self.cfg, 0, 0, 0
        while True:
            yield self.item_wait(item)
            tiles = self.read_item(item)
            if tiles is None:
                yield from self.meet()   # as at the end of the kernel
                return
            yield None
            if not (yield from self.meet()):
                met[0] = True
                return
            self.q[g, warp] = item
            yield None
            self.q_full.arrive()
            for i in range(g, tiles, 2):
                tile = kv + i
                buf, own = tile % c.kv_stages, n & 1
                yield lambda: self.s_full[g][own].test((n >> 1) & 1)
                yield lambda: self.kv_full[buf].test((tile // c.kv_stages) & 1)
                expect(self.scores[g][own].get(warp), ('S', tile), 'scores')
                expect(self.kv[buf], {w: tile for w in range(WARPS)}, 'scales')
                yield None
                if self.rng.random() < 0.5 and i > g:
                    yield lambda: self.pv_done[g].test((n - 1) & 1)
                    want = list(range(kv + g, tile, 2))
                    expect(self.o[g], want, 'sums that are rescaled')
                    yield None
                    expect(self.o[g], want, 'sums at the end of rescaling')
                expect(self.kv[buf], {w: tile for w in range(WARPS)}, 'scales at the end')
                self.scores[g][own] = dict(self.scores[g][own])
                self.scores[g][own][warp] = ('P', tile)
                yield None
                self.p_full[g][own].arrive()
                n += 1
            kv += tiles
            if c.ends_by_item:
                yield lambda: self.item_done.test(item & 1)
            else:   # by the phase of the group's last product
                for other in range(GROUPS):
                    products = (n if other == g else sum((t + 1 - other) // 2 for t in self.work[:item + 1]))
                    if products:
                        yield lambda: self.pv_done[other].test((products - 1) & 1)
            if not (yield from self.meet()):
                met[0] = True
                return
            for when in ('', ' as they are read'):
                for other in range(GROUPS):
                    if tiles > other:
                        expect(self.o[other], list(range(kv - tiles + other, kv, 2)), 'sums of the item' + when)
                yield None
            item += 1


class FewRows(Kernel):
    def __init__(self, stages: int, work: List[int], rng: random.Random, agrees: bool = True, drains: str = ''):
        super().__init__(rng, work, stages, 2, WARPS, WARPS)
        self.agrees = agrees
        self.meeting, self.plain = Meeting(WARPS), Meeting(WARPS)
        self.q: Dict[int, int] = {}
        self.merge: Dict[int, int] = {}
        self.agents = [self.producer(False, drains or drains_in_source('cache_attention.cu'))] + [self.consumer(w) for w in range(WARPS)]

    meet = ManyRows.meet

    @property
    def cfg(self):
        return self   # for meet()

    def consumer(self, warp: int):
        met = [False]
        try:
            yield from self._consumer(warp, met)
        except Aborted:
            if self.agrees and not met[0]:
                yield from self.meet(False)

    def _consumer(self, warp: int, met):
        it = item = 0
        while True:
            yield self.item_wait(item)
            tiles = self.read_item(item)
            if tiles is None:
                yield from self.meet()
                return
            yield None
            if not (yield from self.meet()):
                met[0] = True
                return
            self.q[warp] = item
            yield self.plain.come()[1]
            expect(self.q, {w: item for w in range(WARPS)}, 'queries')
            for _ in range(tiles):
                s = it % self.stages
                yield lambda: self.raw_full[s].test((it // self.stages) & 1)
                expect(self.raw[s], it, 'tile')
                yield None
                expect((self.raw[s], self.q), (it, {w: item for w in range(WARPS)}), 'tile and queries at its end')
                self.raw_empty[s].arrive()
                it += 1
            if not (yield from self.meet()):
                met[0] = True
                return
            self.merge[warp] = item
            yield self.plain.come()[1]
            expect(self.merge, {w: item for w in range(WARPS)}, 'sums')
            yield self.plain.come()[1]
            expect(self.merge, {w: item for w in range(WARPS)}, 'sums as the result is written')
            item += 1
