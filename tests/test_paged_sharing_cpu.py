"""How the serving calls share out their work: host-side rules."""
import math

import pytest
import torch


@pytest.mark.parametrize("hint,keys", [(None, 96), (0, 96), (-3.0, 96), (math.inf, 96), (-math.inf, 96), (math.nan, 96),
                                       (5, 5), (5.25, 6), (0.5, 1), (95.5, 96), (1e30, 96)])
def test_any_hint_of_the_window(ms, hint, keys):
    assert ms.paged._keys_seen(hint, torch.zeros(1, 6, dtype=torch.int32), 16) == keys
