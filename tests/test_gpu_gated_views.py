"""Gated layers over views: no work memory where none is needed, rows of large layers that begin between the places that loads to the LDS can take."""
import pytest
import torch

from test_gpu_gated import Layer, OnDevice

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


# dims whose rows could be loaded to the LDS, in places from which they cannot: a view from the first element on, a stride that no chunk divides; large enough for
# tiles of 256 x 256 wherever they can
@pytest.mark.parametrize("rows,dim,hidden,dtype,pad,first,kept", [
    (4000, 136, 2100, "bfloat16", 1, 1, "as is"), (4000, 136, 2100, "float16", 0, 1, "as is"), (4000, 136, 2100, "bfloat16", 3, 0, "no"), (3000, 72, 2200, "bfloat16", 1, 1, "8 bits"),
    (3001, 132, 2300, "float32", 1, 1, "as is"), (1030, 3600, 4100, "bfloat16", 1, 1, "as is")])
def test_large_layers_over_views(arb, rows, dim, hidden, dtype, pad, first, kept):
    layer = OnDevice(arb, rows, dim, hidden, dtype, kept=kept, pad=pad, first=first, activation="gelu" if rows % 2 else "silu").forward()
    layer.check_forward()
    if kept != "no":
        layer.backward().check_backward()
    layer.check_margins()
