"""The work memory that a gated layer asks for: host code only (the calls that are not refused end at the device, which is not there)."""
import pytest

from test_model_operators_refusals import A, layer, refused


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() != 0:
        pytest.skip("addresses of nothing are for machines without a device")
    return arboretum_amd


# k's shared out, and rows that begin anywhere
@pytest.mark.parametrize("dim,hidden,dtype", [(4096, 64, "float32"), (1001, 64, "bfloat16"), (4095, 16383, "float16")])
def test_few_rows_take_work_only_for_codes(arb, dim, hidden, dtype):
    codes = dict(gate=9 * A, up=10 * A, gate_scales=11 * A, up_scales=12 * A)
    sizes = dict(dim=dim, hidden=hidden, dtype=dtype, w_gate=1 << 40, w_up=1 << 41)
    for rows in (1, 16, 17):
        need = arb.gated_bytes(rows, dim, hidden, dtype=dtype)
        assert need > 0
        if rows <= 16:
            refused(arb, layer, "no HIP device", rows=rows, work=None, work_bytes=0, **sizes)
            refused(arb, layer, "no HIP device", rows=rows, work=None, work_bytes=0, **{**codes, "gate_scales": None, "up_scales": None}, **sizes)
        else:
            refused(arb, layer, "null pointer", rows=rows, work=None, work_bytes=0, **sizes)
        refused(arb, layer, "null pointer", rows=rows, work=None, work_bytes=0, **codes, **sizes)
        refused(arb, layer, "too small: %d bytes" % need, rows=rows, work_bytes=need - 1, **codes, **sizes)
