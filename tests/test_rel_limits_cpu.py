"""CPU: the gradient's limit on bias entries is checked before anything is launched (no device is needed to be refused)."""
import pytest

from vit_amd import _lib

FAKE = 1 << 20


@pytest.mark.parametrize("grid,with_table", [((1, 15872), True), ((89, 89), True), ((1, 16384), True), ((1, 16384), False), ((128, 128), False)])
def test_gradient_is_refused_before_its_first_launch(grid, with_table):
    lib = _lib.load()
    p = _lib.vit_rel_pos(prefix=0, grid_h=grid[0], grid_w=grid[1], num_buckets=(2 * grid[0] - 1) * (2 * grid[1] - 1))
    # (a workspace of no size: without the limit's check the call would end at that one)
    assert lib.vit_attention_rel_bwd(p, FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE if with_table else None, FAKE, 0, 1, 1, 1, 16, 0.25,
                                     None) == -1
    assert b"bias entries" in lib.vit_last_error()
