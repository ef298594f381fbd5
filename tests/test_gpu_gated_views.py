"""Gated layers over views: no work memory where none is needed."""
import pytest
import torch

from test_gpu_gated import Layer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,dim,hidden", [(1, 4096, 64), (16, 1001, 64), (7, 513, 200)])
def test_few_rows_without_work_memory(arb, rows, dim, hidden, dtype):
    with_work, without = (Layer(arb, rows, dim, hidden, dtype) for _ in range(2))
    with_work.forward()
    without.arb.gated(without.out.data_ptr(), without.d_x.data_ptr(), without.d_wg.data_ptr(), without.d_wu.data_ptr(), rows, dim, hidden, None, 0, gate=without.gate.data_ptr(),
                      up=without.up.data_ptr(), dtype=dtype)
    without.check_forward()
    for name in ("out", "gate", "up"):
        assert torch.equal(getattr(with_work, name), getattr(without, name))
