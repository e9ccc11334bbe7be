"""The barrier protocols of the kernels of attention over the quantized cache, model-checked on the host under random schedules (no GPU)."""
import dataclasses
import random

import pytest

from cache_attention_model import FewRows, ManyRows, many_rows_config_from_source
from pipeline_model import ProtocolError

WORK = [[1], [2], [3], [1, 1, 1, 1, 1], [2, 1, 3, 2, 1], [40], [1, 9, 2, 8, 1, 7], [4, 4, 4, 4, 4, 4, 4], []]


@pytest.mark.parametrize('work', WORK, ids=str)
def test_many_rows_under_random_schedules(work):
    cfg = many_rows_config_from_source()
    for seed in range(40):
        for delay in (0.2, 0.9, 0.99):
            ManyRows(cfg, work, random.Random(seed)).run(copy_delay=delay)


def runs_out(make, agents, seeds):
    """Schedules in which the n-th blocked wait of each role runs out; in how many one did."""
    runs = 0
    for seed in range(seeds):
        for agent in range(agents):
            for nth in (1, 2, 3, 17):
                kernel = make(seed)
                kernel.expire = (agent, nth)
                kernel.run(copy_delay=(0.9, 0.99, 0.999)[seed % 3])
                runs += any(kernel.abort)
    return runs


@pytest.mark.parametrize('work', [[2], [1, 2, 1, 3], [9, 3], [2, 2, 2, 2, 2]], ids=str)
def test_a_wait_of_the_kernel_for_many_rows_that_runs_out_ends_every_role(work):
    """The other roles' waits end by the flag, warps that meet at the named barrier leave there together, and nothing is on its way when the CTA ends."""
    cfg = many_rows_config_from_source()
    assert runs_out(lambda seed: ManyRows(cfg, work, random.Random(seed)), 2 + 4 + 8, 12) > 50


@pytest.mark.parametrize('stages', [2, 3, 6])
@pytest.mark.parametrize('work', WORK, ids=str)
def test_few_rows_under_random_schedules(stages, work):
    for seed in range(30):
        for delay in (0.2, 0.9, 0.99):
            FewRows(stages, work, random.Random(seed)).run(copy_delay=delay)


@pytest.mark.parametrize('work', [[2], [1, 2, 1, 3], [9, 3], [2, 2, 2, 2, 2]], ids=str)
def test_a_wait_of_the_kernel_for_few_rows_that_runs_out_ends_every_role(work):
    assert runs_out(lambda seed: FewRows(3, work, random.Random(seed)), 1 + 4, 25) > 50


def found(make, expire=None, seeds=60, what='', delay=0.9):
    errors = 0
    for seed in range(seeds):
        kernel = make(seed)
        if expire:
            kernel.expire = expire(seed)
        try:
            kernel.run(copy_delay=delay)
        except ProtocolError as e:
            assert what in str(e), e
            errors += 1
    return errors


def test_the_models_find_what_would_be_wrong():
    cfg = many_rows_config_from_source()
    many = lambda work, **change: lambda seed: ManyRows(dataclasses.replace(cfg, **change), work, random.Random(seed))
    # scores asked for so far ahead that they would take the place of probabilities (or that the ring has no room for them)
    assert found(many([12], ahead=4)) > 0
    # the end of an item by a barrier of which two phases may be under way
    assert found(many([5, 5], ends_by_item=False), seeds=3000, delay=0.2) > 0
    # warps that leave one by one, with the others at the named barrier
    assert found(many([1, 2, 3], agrees=False), lambda seed: (6 + seed % 8, 1 + seed // 8), 200, 'deadlock', 0.5) > 0
    assert found(lambda seed: FewRows(3, [1, 2, 3], random.Random(seed), agrees=False), lambda seed: (1 + seed % 4, 1 + seed // 8), 200, 'deadlock', 0.5) > 0
    # copies or products on their way when the CTA ends: the copying warp may be through when another's wait runs out
    for drains, agent, work in (('never', 0, [9]), ('never', 1, [9]), ('own', 2, [2])):
        assert found(many(work, drains=drains), lambda seed: (agent, 1 + seed % 3), 300, 'retired with', 0.999) > 0
        assert found(lambda seed: FewRows(3, work, random.Random(seed), drains=drains), lambda seed: (agent, 1 + seed % 3), 100, 'retired with', 0.99) > 0
