"""GPU: the ends of what attention over groups takes -- sinks and windows up to the type's
largest.

Attention is held to the tolerances of test_gpu_groups.py."""
import pytest
import torch
from test_gpu_groups import check_groups, make_groups

pytestmark = pytest.mark.gpu

LARGEST = 2 ** 31 - 1


@pytest.mark.parametrize("window,sinks", [(1, LARGEST), (1, LARGEST - 20), (9, 2 ** 30), (LARGEST, 0), (LARGEST, LARGEST), (2 ** 30, 1)])
def test_sinks_and_windows_of_any_size(ufb, dev, window, sinks):
    """Groups that share little or nothing, whose streams lie together in a tile: a stream's first own key is
    then behind the tile's, and its keys are counted from there."""
    for page, dim, group in ((16, 64, 3), (64, 128, 40)):
        cache, lengths, sizes = make_groups(ufb, dev, [(0, [20, 40, 9, 300]), (130, [5, 5, 90])], 2, dim, page)
        for counts in ([1] * 7, [4, 30, 9, 200, 2, 5, 1]):
            for causal in (True, False):
                check_groups(ufb, cache, list(range(7)), counts, sizes, 2 * group, torch.float16, window=window, sinks=sinks,
                             causal=causal)
