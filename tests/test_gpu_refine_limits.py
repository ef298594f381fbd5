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


def sums_64(leaf, w, classes):
    """Sums of leaf weights, and of their magnitudes: [classes][rows].  Tree t is of class t % classes."""
    sums, size = np.zeros((classes, leaf.shape[1])), np.zeros((classes, leaf.shape[1]))
    for t in range(len(leaf)):
        sums[t % classes] += w[t][leaf[t]]
        size[t % classes] += np.abs(w[t][leaf[t]])
    return sums, size


@pytest.mark.parametrize("objective,classes", [(0, 1), (1, 1), (4, 3), (3, 2)])
def test_several_steps_of_every_objective(arb, objective, classes):
    """Against 64 bits, the error carried from step to step.  With e the error of the weights so far (per leaf), a sum of a row's
    weights is off by the e of its leaves and by (trees + 3) u of their magnitudes, and a direction by no more than that (the slopes of the links are at
    most 1; of the soft-max, by the largest over the classes, twice) and 8 u of values around 1.  A gradient sums these over its rows and
    is off by (rows + 4) u of the magnitudes besides.  The moments take such an error on with their factors and 5 and 8 roundings; the step
    size m / (sqrt(v) / root + eps) is off by size (dm / den + |m| dr / den^2) and 13 roundings, dr = dv / (sqrt(v) root) or
    sqrt(dv) / root, the lesser.  With eps = 0.05, large against most gradients, this stays small."""
    from test_gpu_refine import U, directions_64, walk
    model, data, X, y, labels = make(arb, objective, classes=classes, rounds=4, rows=2000)
    n, trees, steps, lr, eps, decay, b1, b2 = len(X), model.num_trees(), 5, 0.02, 0.05, 0.1, 0.8, 0.9
    init = {0: 0.5, 1: 0.0}.get(objective, 0.0)
    leaf = walk(model, X)
    w = np.array([model.tree(t)["weights"] for t in range(trees)], np.float64)
    e, m, v, dm, dv = (np.zeros_like(w) for _ in range(5))
    before = w.copy()
    for step in range(1, steps + 1):
        sums, size = sums_64(leaf, w, classes)
        off, _ = sums_64(leaf, e, classes)
        d = directions_64(objective, sums, init, y, labels)
        dd = 2 * (off + (trees // classes + 3) * U * (size + off)).max(0) + 8 * U * (1 + np.abs(sums).max(0) + np.abs(d).max(0))
        for t in range(trees):
            g, dg, mag = (np.zeros(w.shape[1]) for _ in range(3))
            np.add.at(g, leaf[t], -d[t % classes] / n)
            np.add.at(dg, leaf[t], dd / n)
            np.add.at(mag, leaf[t], np.abs(d[t % classes]) / n)
            dg += (np.bincount(leaf[t], minlength=len(g)) + 4) * U * (mag + dg)
            dm[t] = b1 * dm[t] + (1 - b1) * dg + 5 * U * (b1 * np.abs(m[t]) + (1 - b1) * np.abs(g))
            dv[t] = b2 * dv[t] + (1 - b2) * (2 * np.abs(g) + dg) * dg + 8 * U * (b2 * v[t] + (1 - b2) * g * g)
            m[t], v[t] = b1 * m[t] + (1 - b1) * g, b2 * v[t] + (1 - b2) * g * g
            root, factor = np.sqrt(1 - b2 ** step), lr / (1 - b1 ** step)
            den = np.sqrt(v[t]) / root + eps
            dr = np.minimum(np.sqrt(dv[t]), dv[t] / np.maximum(np.sqrt(v[t]), 1e-300)) / root
            moved = factor * m[t] / den
            at = np.abs(w[t])
            # (the denominator of the other side is no less than eps)
            e[t] = e[t] * (1 - lr * decay) + 1.01 * factor * (dm[t] / den + np.abs(m[t]) * dr / (den * eps)) + 14 * U * np.abs(moved) + 3 * U * at
            w[t] = w[t] * (1 - lr * decay) - moved
    model.refine_leaves(steps=steps, lr=lr, eps=eps, weight_decay=decay, beta1=b1, beta2=b2)
    got = weights(model).reshape(w.shape).astype(np.float64)
    assert (np.abs(got - w) <= e).all()
    # the bound tells a wrong step from a right one: it is far below what a weight moves
    assert np.median(e) < 1e-3 * np.abs(w - before).max()
