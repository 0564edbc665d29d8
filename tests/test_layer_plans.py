"""Forced plans of products, on the host."""
import pytest

from mini_nangila_b200 import _ext

pytestmark = pytest.mark.skipif(not _ext.cuda_available(), reason="the CUDA extension is not built")


@pytest.mark.parametrize("k,dual,fp8", [(8, 0, False), (64, 0, False), (65, 0, False), (200, 1, False), (512, 2, False),
                                        (130, 3, False), (128, 0, True), (300, 1, True)])
def test_a_forced_plan_gives_each_piece_of_k_a_block(k, dual, fp8):
    """A piece without a block of k has no product, and what its tensor memory
    holds from before would be joined as its sums."""
    ext = _ext.cuda()
    blocks = -(-k // (128 if fp8 else 64)) * (2 if dual == 2 else 1)
    try:
        for splits in (1, 2, 3, 64):
            ext.dense_force_plan(1, 128, splits)
            assert ext.dense_plan(300, 500, k, dual, fp8, 148) == [1, 128, min(splits, blocks)]
    finally:
        ext.dense_force_plan(0, 0, 0)
