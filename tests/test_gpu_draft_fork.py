"""Forks whose pages meet those of other pairs."""
import pytest

from .test_gpu_draft_layers import check_fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [1, 28])
def test_a_page_that_another_pair_copies_from_is_refused(cuda_device, layers):
    """Pair 0 would write what pair 1 reads: it is left undone, pair 1 is done."""
    dev, lens = cuda_device, [20, 48, 30, 0, 0, 0]

    def last_of(b):
        return lambda free, table: [int(table[b, (lens[b] - 1) // 16]), free[0]]

    check_fork(dev, lens, [(0, 3), (2, 4)], pages=last_of(2), bad="fork", undone=(0,), layers=layers)
    check_fork(dev, lens, [(0, 3), (2, 4), (2, 5)], pages=lambda free, table: [int(table[2, 1]), *free[:2]], bad="fork",
               undone=(0,), layers=layers)
    # each other's
    check_fork(dev, lens, [(0, 3), (2, 4)], pages=lambda free, table: [int(table[2, 1]), int(table[0, 1])], bad="fork",
               undone=(0, 1), layers=layers)
    # far apart in a long list
    lens = [20] * 400 + [0] * 400
    pairs = [(b, 400 + b) for b in range(400)]
    check_fork(dev, lens, pairs, pages=lambda free, table: [int(table[399, 1])] + free[1:400], bad="fork", undone=(0,),
               layers=layers)


def test_a_page_that_no_pair_copies_from(cuda_device):
    """The last page of a source that ends with it is shared, not copied; of a place without a pair nothing is looked at."""
    dev, lens = cuda_device, [20, 48, 30, 0, 0, 0]
    check_fork(dev, lens, [(0, 3), (-1, 4), (2, -1)], pages=lambda free, table: [free[0], free[1], free[2]], undone=(1, 2))
    check_fork(dev, lens, [(1, 3), (0, 4)], pages=lambda free, table: [int(table[0, 1]), free[0]])


@pytest.mark.parametrize("layers", [1, 28])
def test_a_page_that_only_one_pair_needs(cuda_device, layers):
    """Sources that end with a page need none: what stands in their places, the same page as another's, is not looked at."""
    dev, lens = cuda_device, [20, 48, 30, 0, 0, 0, 0]
    check_fork(dev, lens, [(0, 4), (1, 5)], pages=lambda free, table: [free[0], free[0]], layers=layers)
    check_fork(dev, lens, [(1, 4), (3, 5), (2, 6)], pages=lambda free, table: [free[0]] * 3, layers=layers)
    check_fork(dev, lens, [(1, 4), (0, 5), (2, 6)], pages=lambda free, table: [free[0]] * 3, bad="fork", undone=(1, 2),
               layers=layers)
