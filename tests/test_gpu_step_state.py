"""The state that si_kv_step takes: what no step left is refused, and a refused step leaves
everything as it was, in each of the kernel's forms (one small workgroup; one large; several with
the new state over the old; several with it beside the old)."""
import numpy as np
import pytest

from tests.gpu_helpers import dev, torch_cuda
from tests.test_gpu_step import Tables, filled, host

pytestmark = pytest.mark.gpu

# sequences and max_rows that take each form, and whether the new state lies beside the old
FORMS = [(3, 40, False), (300, 1200, False), (700, 3000, False), (700, 3000, True)]


class Fleet:
    """Tables whose first sequences are looked at; the others have no rows."""

    def __init__(self, form, page=4, max_pages=8, window=4, sinks=0, npages=40):
        self.nseq, max_rows, self.apart = form
        self.t = Tables(self.nseq, page, npages, max_pages, max_rows, window, sinks, seed=2)

    def all(self, first):
        x = np.zeros(self.nseq, np.int32)
        x[:len(first)] = first
        return x

    def step(self, have, add):
        """The step's code, and whether lists, ring and state are as they were."""
        t = self.t
        before = [host(x).copy() for x in (t.pages, t.ring, t.free, t.held)]
        free, held = (x.clone().fill_(-7) for x in (t.free, t.held)) if self.apart else (None, None)
        t.run(dev(self.all(have)), dev(self.all(add)), free, held)
        if self.apart:
            t.free, t.held = free, held
        after = [host(x) for x in (t.pages, t.ring, t.free, t.held)]
        return int(host(t.status)[0]), all(np.array_equal(a, b) for a, b in zip(before, after))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sinks,lowest", [(0, 15), (3, 15), (6, 15)])
def test_tables_positions_behind_those_given_back(form, sinks, lowest):
    """A have whose rows would see, or be written to, pages that were given back: refused, down to
    the lowest at which these still lie behind the window."""
    f = Fleet(form, sinks=sinks)
    assert f.step([0, 0, 0], [18, 4, 1]) == (0, False)
    # of 18 positions 0 to 14 lie behind: three pages, but the sinks'
    kept = -(-sinks // 4)
    assert f.step([18, 4, 1], [0, 1, 0]) == (0, False)
    assert host(f.t.held)[0].tolist() == [5, 3 - kept]
    for have in (lowest - 1, 5, 1, 0):
        assert f.step([have, 5, 1], [5, 1, 0]) == (4, True)
        assert (host(f.t.slot) == -1).all() and (host(f.t.start) == 0).all()
    assert f.step([lowest, 5, 1], [3, 1, 0])[0] == 0


@pytest.mark.parametrize("form", FORMS)
def test_tables_refused_step_says_what_it_was_given(form):
    """The contexts of a refused step are its have, of sequences that end too, so that the next
    step, made from them, ends them."""
    f = Fleet(form)
    assert f.step([0, 0, 0], [18, 4, 2])[0] == 0
    assert f.step([18, 4, 2], [1, 1, 1])[0] == 0
    held = host(f.t.held).copy()
    assert f.step([-1, 5, -3], [0, 28, 0]) == (4, True)
    assert host(f.t.ctx)[:3].tolist() == [-1, 5, -3]
    assert np.array_equal(host(f.t.held), held)
    assert f.step(host(f.t.ctx)[:3], [0, 2, 0])[0] == 0
    assert host(f.t.held)[:3].tolist() == [[0, 0], [2, 0], [0, 0]]
    assert int(host(f.t.free)[1]) == 40 - 2


@pytest.mark.parametrize("form", FORMS)
def test_tables_more_pages_than_the_pool(form):
    """A ring and lists that together hold more ids than there are would hand out a page twice:
    refused, also where nothing is given back."""
    f = Fleet(form)
    assert f.step([0, 0, 0], [7, 4, 1])[0] == 0  # four pages
    begin = int(host(f.t.free)[0])
    for count in (37, 40):
        f.t.free.copy_(dev(np.array([begin, count], np.int32)))
        for add in ([1, 0, 0], [0, 1, 0]):
            assert f.step([7, 4, 1], add) == (4, True)
    f.t.free.copy_(dev(np.array([begin, 36], np.int32)))
    assert f.step([7, 4, 1], [0, 1, 0])[0] == 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("held", [(9, 0), (-1, 0), (2, -1), (2, 3), (2 ** 31 - 1, 0), (0, 1),
                                  (-2 ** 31, 2 ** 31 - 1)])
@pytest.mark.parametrize("ends", [False, True])
def test_tables_counts_that_no_step_left(form, held, ends):
    """Pages taken or given back that cannot be: refused, and left as they are."""
    f = Fleet(form)
    assert f.step([0, 0, 0], [7, 4, 1])[0] == 0
    h = host(f.t.held).copy()
    h[1] = held
    f.t.held.copy_(dev(h))
    for _ in range(2):
        assert f.step([7, -1 if ends else 0, 1], [0, 0, 0]) == (4, True)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("free", [(40, 3), (-1, 3), (5, -1), (5, 41), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_tables_ring_that_no_step_left(form, free):
    """A ring whose numbers cannot be: refused, and empty from then on, so that none of its ids
    is handed out."""
    f = Fleet(form)
    assert f.step([0, 0, 0], [7, 4, 0])[0] == 0
    kept = [host(x).copy() for x in (f.t.pages, f.t.ring, f.t.held)]
    f.t.free.copy_(dev(np.array(free, np.int32)))
    assert f.step([7, 4, 0], [1, 0, 0]) == (4, False)
    assert host(f.t.free).tolist() == [0, 0]
    for a, b in zip(kept, (f.t.pages, f.t.ring, f.t.held)):
        assert np.array_equal(a, host(b))
    assert f.step([7, 4, 0], [0, 0, 1])[0] == 2


def test_tables_whole_pool_held():
    """Lists that hold every page of the pool, in place and full: no row more, but a step without
    one, and one that ends a sequence."""
    torch_cuda()
    t, have = filled(npages=4)
    for h, a, code in (([2, 2, 2, 2], [2, 2, 2, 2], 0), ([4, 4, 4, 4], [0, 0, 0, 1], 2),
                       ([4, -1, 4, 4], [0, 0, 0, 0], 0), ([4, 0, 4, 4], [0, 0, 0, 1], 0)):
        t.run(dev(np.array(h, np.int32)), dev(np.array(a, np.int32)))
        assert host(t.status)[0] == code
    assert host(t.free)[1] == 0
