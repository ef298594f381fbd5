"""A booster's log probabilities are the same wherever the rows are: bin ids on the host, in the caller's blocks, blocks that end inside a row of workgroups."""
import numpy as np
import pytest
import torch  # noqa: F401  (its runtime before the package's)

from test_gpu_blocks import to_block
from test_gpu_refine import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


@pytest.mark.parametrize("rows,block_rows", [(1000, 4096), (5000, 1024), (70_000, 65_536)])
def test_rows_in_blocks(arb, rows, block_rows):
    classes = 5
    model, data, X, _, labels = make(arb, 3, rows=rows, rounds=3, classes=classes, prebinned=True)
    bins = X.astype(np.uint8)
    blocks = [to_block(bins[b:b + block_rows], block_rows) for b in range(0, rows, block_rows)]
    in_blocks = arb.DMatrix.from_blocks([b.ptr for b in blocks], block_rows, rows, bins.shape[1], labels=labels)
    want = model.log_probs(data, top=4)
    for other in (in_blocks, arb.DMatrix(X, labels=labels)):  # (bin ids as floats walk the same way)
        got = model.log_probs(other, top=4)
        assert sorted(got) == sorted(want) and all(np.array_equal(got[k], want[k]) for k in want)
