"""What a refinement leaves alone, keeps to or refuses once there are trees."""
import numpy as np
import pytest

from test_gpu_refine import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


def weights(model):
    return np.concatenate([model.tree(t)["weights"] for t in range(model.num_trees())])


def test_a_loaded_booster_of_several_classes_stays_as_it_was(arb):
    model, data, _, _, _ = make(arb, 4, classes=3, rounds=4)
    other = arb.load(model.dump())
    before, answer = weights(other), other.predict(data)
    with pytest.raises(arb.ArboretumError, match="as many trees of each class"):
        other.refine_leaves(data, steps=3)
    other.data = data
    other.grow_tree()  # nor with trees of its own behind the loaded ones
    with pytest.raises(arb.ArboretumError, match="as many trees of each class"):
        other.refine_leaves(steps=3)
    assert np.array_equal(weights(other)[:len(before)], before) and np.array_equal(other.predict(data, 12), answer)
    model.refine_leaves(steps=3)
    assert not np.array_equal(weights(model), before)
