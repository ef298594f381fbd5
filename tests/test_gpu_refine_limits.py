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


def test_a_refinement_that_diverges_leaves_the_booster_as_it_was(arb):
    # the weights of a leaf move by 2e37 a step, and the sum of twenty is beyond float32
    model, data, _, _, _ = make(arb, 0, rounds=20)
    before, answer = weights(model), model.predict(data)
    with pytest.raises(arb.ArboretumError, match="not finite"):
        model.refine_leaves(lr=2e37, steps=6)
    assert np.array_equal(weights(model), before) and np.array_equal(model.predict(data), answer)
    model.grow_tree()
    model.refine_leaves(steps=2)
    assert np.isfinite(weights(model)).all()


def test_leaves_that_no_row_reaches_stay_where_they_are(arb):
    model, data, X, y, _ = make(arb, 0, rounds=5, depth=5)
    some = slice(0, 60)
    for eps in (0.0, 1e-50):
        with pytest.raises(arb.ArboretumError, match="eps must be at least"):
            model.refine_leaves(arb.DMatrix(X[some], y=y[some]), steps=2, eps=eps)
    from test_gpu_refine import walk
    leaf, before = walk(model, X[some]), weights(model).reshape(5, -1)
    model.refine_leaves(arb.DMatrix(X[some], y=y[some]), steps=3, eps=2.0 ** -126)
    after = weights(model).reshape(5, -1)
    for t in range(5):
        reached = np.isin(np.arange(before.shape[1]), leaf[t])
        assert not reached.all() and np.array_equal(after[t][~reached], before[t][~reached])
        assert np.isfinite(after[t]).all() and (after[t][reached] != before[t][reached]).any()
