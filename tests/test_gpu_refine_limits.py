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


@pytest.mark.parametrize("objective,classes", [(0, 1), (1, 1), (4, 3)])
def test_refined_weights_keep_to_the_largest_leaf_weight(arb, objective, classes):
    # a grown leaf is at most max_leaf_weight * eta, the product rounded to float32
    most = np.float32(0.3) * np.float32(0.5)
    config = {"objective": objective, "method": 1, "internals": {"hist_size": 64, "double_precision": True},
              "tree": {"max_depth": 4, "eta": 0.5, "max_leaf_weight": 0.3, "lambda": 1.0, "min_child_weight": 1.0}}
    if classes > 1:
        config["tree"]["labels_count"] = classes
    _, _, X, y, labels = make(arb, objective, classes=classes, rounds=1)
    data = arb.DMatrix(X, y=y, labels=labels)
    model = arb.train(config, data, 4)
    model.synchronize()
    grown = weights(model)
    assert np.abs(grown).max() <= most
    lr = 0.01
    model.refine_leaves(steps=40, lr=lr)
    refined = weights(model)
    assert not np.array_equal(refined, grown)
    assert np.abs(refined).max() == most  # (leaves that would go on are held there)
    # without the limit the same steps go beyond it
    free = arb.train(dict(config, tree=dict(config["tree"], max_leaf_weight=0.0)), data, 4)
    free.refine_leaves(steps=40, lr=lr)
    assert np.abs(weights(free)).max() > most


def test_steps_within_a_largest_leaf_weight_are_the_operators_and_the_limit_in_turn(arb):
    import torch
    from test_gpu_refine import tokens_of
    most = np.float32(0.2) * np.float32(0.3)
    _, _, X, y, _ = make(arb, 0, rounds=1)
    config = {"objective": 0, "method": 1, "internals": {"hist_size": 64},
              "tree": {"max_depth": 4, "eta": 0.3, "max_leaf_weight": 0.2, "lambda": 1.0}}
    data = arb.DMatrix(X, y=y)
    model = arb.train(config, data, 6)
    n, trees, steps, lr = len(X), 6, 9, 0.02
    held, (leaves,) = tokens_of(arb, model, data)
    w = torch.tensor(weights(model)).cuda()
    grad, m, v = torch.empty_like(w), torch.zeros_like(w), torch.zeros_like(w)
    out, target = torch.empty(n, device="cuda"), torch.tensor(y).cuda()
    pairs = torch.empty(2, n * trees, dtype=torch.int32, device="cuda")
    size = max(arb.embedding_sort_bytes(n, leaves, bag=trees), arb.embedding_grad_bytes(n, 1, bag=trees))
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    arb.embedding_sort(pairs[0].data_ptr(), pairs[1].data_ptr(), held.data_ptr(), n, leaves, work.data_ptr(), size, bag=trees,
                       token_stride=1, bag_stride=n)
    for step in range(1, steps + 1):
        arb.embedding(out.data_ptr(), w.data_ptr(), held.data_ptr(), n, leaves, 1, bag=trees, token_stride=1, bag_stride=n)
        d = target - (out + 0.5)
        arb.embedding_grad(grad.data_ptr(), d.data_ptr(), pairs[0].data_ptr(), pairs[1].data_ptr(), n, leaves, 1, work.data_ptr(),
                           size, bag=trees, scale=-1.0 / n)
        arb.adamw([w.data_ptr()], [grad.data_ptr()], [m.data_ptr()], [v.data_ptr()], [leaves], step, lr, weight_decay=0.0)
        w.clamp_(-float(most), float(most))
    model.refine_leaves(steps=steps, lr=lr)
    assert np.array_equal(weights(model), w.cpu().numpy())
    assert (np.abs(weights(model)) == most).any()


def test_a_limit_of_0_holds_every_leaf(arb):
    _, _, X, y, _ = make(arb, 0, rounds=1)
    model = arb.train({"objective": 0, "method": 1, "internals": {"hist_size": 64},
                       "tree": {"max_depth": 3, "eta": 0.0, "max_leaf_weight": 0.2}}, arb.DMatrix(X, y=y), 2)
    model.refine_leaves(steps=3)
    assert not weights(model).any()
