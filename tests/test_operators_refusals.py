"""More calls that the tensor operators refuse, each of which would be answered wrongly: host code only, so nothing here
reaches a GPU (addresses are never followed: every call is refused before a kernel is launched)."""
import pytest

from test_operators_host import A, adamw


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    return arboretum_amd


@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-46, 1e-39])
def test_adamw_refuses_an_eps_that_float32_does_not_hold(arb, eps):
    # an element whose gradient has always been 0, a table's row that no token names, would become 0 / 0
    with pytest.raises(arb.ArboretumError, match="eps must be at least 2\\^-126"):
        adamw(arb, eps=eps)


@pytest.mark.parametrize("change", [dict(lr=1e300), dict(lr=1e38), dict(lr=1e30, weight_decay=1e30), dict(eps=1e39), dict(grad_scale=-1e39),
                                    dict(grad_scale=1e300)])
def test_adamw_refuses_constants_beyond_float32(arb, change):
    # (1e38 / (1 - 0.9): the step's factor, which a moment of 0 would meet)
    with pytest.raises(arb.ArboretumError, match="beyond float32"):
        adamw(arb, **change)


def test_adamw_refuses_constants_beyond_float32_whatever_the_device_words_replace(arb):
    with pytest.raises(arb.ArboretumError, match="beyond float32"):
        adamw(arb, grad_scale=1e39, lr_device=A, step_device=A)
    with pytest.raises(arb.ArboretumError, match="eps must be at least"):
        adamw(arb, eps=0.0, lr_device=A, step_device=A)
