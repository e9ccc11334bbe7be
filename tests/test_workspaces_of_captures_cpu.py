"""A graph has scratch of its own, and nothing is kept for graphs that nobody captured; with the stand-ins of test_workspaces_cpu."""
import weakref

from test_workspaces_cpu import DEVICE, SIZE, Workspaces, told  # noqa: F401 (told: a fixture)


def test_captures_share_nothing_with_each_other_nor_with_calls_outside(told):
    w = Workspaces()
    outside = w.during(0)
    first, keep = w.during(1), w._buffers[(0, 77)]
    again = w.during(1)
    second, keep2 = w.during(2), w._buffers[(0, 77)]
    assert first == again and len({outside, first, second}) == 3 and keep is not keep2
    assert w.during(0) == outside and told[77] == outside     # their own again
    assert w.during(3) not in (0, outside)


def test_a_capture_that_asks_for_more(told):
    w = Workspaces()
    small, large = w.during(1), w.during(1, 8 * SIZE)
    assert w.during(1) == large and w.during(0, SIZE) != large
    outside = w.during(0)
    assert w.during(2) != outside and w.during(0) == outside and small


def test_what_calls_outside_outgrow_is_given_back(told):
    w = Workspaces()
    gone = []
    for size in (SIZE, 2 * SIZE, 4 * SIZE, 8 * SIZE):
        w.during(0, size)
        gone.append(weakref.ref(w._buffers[(0, 77)]))
        if size == 2 * SIZE:
            w.during(5)   # a capture in between holds nothing of it
            w.during(0)
    assert [r() is None for r in gone] == [True, True, True, False]
    w.swap(DEVICE, 77, None)
    assert gone[-1]() is None


def test_a_graph_that_owns_its_warm_up_captures_with_it(told):
    """As CudaGraph does: the stream's scratch is taken out, made anew by the warm-up, and taken away with the graph."""
    w = Workspaces()
    around = w.during(0)
    before = w.swap(DEVICE, 77, None, exclusive=True)
    warm = w.during(0)
    assert w.during(4) == warm
    larger = w.during(4, 4 * SIZE)         # the warm-up did less: the graph has both
    held = w.swap(DEVICE, 77, before)
    assert held.data_ptr() == larger and w.outside(held).data_ptr() == warm
    assert w.during(0) == around and told[77] == around
    assert w.during(6) not in (around, warm, larger)   # no longer exclusive
