"""The paged 8-bit cache at the ends of what its calls accept."""
import numpy as np
import pytest
import torch

from paged_cases import Cache, check, expected
from test_gpu_paged_attention import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30])
@pytest.mark.parametrize("max_new", [None, 64])  # the kernel of few rows, that of many
def test_windows_that_hide_nothing(cuda, window, max_new):
    """Windows up to the largest 32-bit number, with more rows than tokens: rows before the
    first token see nothing, the others everything before them."""
    c = Cache([3, 40, 0, 131], kind="e4m3", seed=21)
    new, G = [6, 2, 4, 1], 3
    q = c.queries(new, G)
    out, ml = run(cuda, c, q, new, G, window=window, max_new=max_new)
    e_out, e_ml, b_out, b_ml = expected(c, q, new, G)
    assert (out[:3] == 0).all() and np.isneginf(ml[:3, :, 0]).all()
    check(out, e_out, b_out, "out")
    check(ml, e_ml, b_ml, "ml")
