"""How the serving calls share out their work: host-side rules."""
import math

import pytest
import torch


@pytest.mark.parametrize("hint,keys", [(None, 96), (0, 96), (-3.0, 96), (math.inf, 96), (-math.inf, 96), (math.nan, 96),
                                       (5, 5), (5.25, 6), (0.5, 1), (95.5, 96), (1e30, 96)])
def test_any_hint_of_the_window(ms, hint, keys):
    assert ms.paged._keys_seen(hint, torch.zeros(1, 6, dtype=torch.int32), 16) == keys


def test_no_workspace_where_nothing_is_shared_out(ms):
    """As many (sequence, head) pairs as CTAs, or more: a CTA each and no sums to
    join."""
    import ctypes
    L = ms._lib

    def need(B, H, num_ctas):
        a = L.TreeArgs(dtype=L.BF16, cache_dtype=L.I8, B=B, H=H, D=64, n=3, num_ctas=num_ctas)
        return L.load().screen_tree_workspace_size(ctypes.byref(a))

    assert need(4, 16, 592) >= 592 * 3 * 64 * 4
    assert need(4, 16, 1) == need(4, 16, 64) == need(40, 16, 592) == need(37, 16, 60000) == 0
    assert ms.paged._tree_ctas(64, 10000) > 1 and ms.paged._tree_ctas(640, 10000) == 1
    assert ms.paged._tree_ctas(64, 100) == 1


