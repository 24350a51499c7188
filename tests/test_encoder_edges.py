"""Corners of the read encoder's operators that tests/test_encoder_ops.py does not reach; the definitions in 64
bits and the tolerances are those of that file."""
import pytest
import torch

from test_encoder_ops import BF16, F16, check_device, linear_check, linear_inputs, ops


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,act", [(20000, 64, 517, "gelu"), (13331, 40, 1279, "relu"), (40001, 24, 333, "gelu")])
def test_gradient_of_odd_widths_whose_last_tile_is_half_empty(m, k, n, act):
    """Rows that no TMA can read, on SM pairs of which the last one's second half has no rows (m mod 256 in
    1..128): that half stores nothing for its tile, and the staging buffers of the tiles around it are
    still waited for.  A buffer taken too early shows in one call of many, so calls repeat bit for bit."""
    x, w, b, _, g = linear_inputs(m, k, n, F16, seed=m)
    assert 1 <= m % 256 <= 128 and n % 8
    linear_check(x, w, b, None, act, g * 0.05)
    first = ops().linear_backward(g, x, w, b, act, True, True, True)
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(first, ops().linear_backward(g, x, w, b, act, True, True, True)))
    check_device()
