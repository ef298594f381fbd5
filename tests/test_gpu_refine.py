"""Leaf tokens and the refinement of leaf weights: the booster's own path over the embedding operators.

Bounds of a first step.  From zero states AdamW's first step is lr g / (|g| + eps), whose derivative by g is at most
1 / eps; a gradient that is off by dg moves a weight by at most lr dg / eps, and the step's own roundings (13 of 2^-24, see
the tests of the operators) by 13 u lr, the weight's by u |w| each for decay and difference."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def arb():
    import arboretum_amd
    if arboretum_amd.device_count() < 1:
        pytest.fail("no HIP device")
    return arboretum_amd


def make(arb, objective, rows=3000, features=9, rounds=7, depth=4, classes=1, missing=0.1, seed=0, prebinned=False):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(rows, features)).astype(np.float32)
    score = X[:, 0] * X[:, 1] + X[:, 2] + 0.3 * rng.normal(size=rows)
    X[rng.random(X.shape) < missing] = np.nan
    if prebinned:
        X = np.clip(np.nan_to_num(X, nan=4.0) * 8 + 32, 0, 63).astype(np.uint8)
    y, labels = None, None
    if classes > 1:
        labels = np.digitize(score, np.quantile(score, np.arange(1, classes) / classes)).astype(np.uint8)
    else:
        y = (score > 0).astype(np.float32) if objective == 1 else score.astype(np.float32)
    config = {"objective": objective, "method": 1, "internals": {"hist_size": 64, "double_precision": True},
              "tree": {"max_depth": depth, "eta": 0.3, "lambda": 1.0, "min_child_weight": 1.0}}
    if classes > 1:
        config["tree"]["labels_count"] = classes
    data = arb.DMatrix(X, y=y, labels=labels, quantized=prebinned)
    model = arb.train(config, data, rounds)
    model.synchronize()
    return model, data, X.astype(np.float32), y, labels


def walk(model, X):
    """The leaf of every row in each tree, [trees][rows]."""
    out = []
    for t in range(model.num_trees()):
        tree = model.tree(t)
        nodes = len(tree["fid"])
        at = np.zeros(len(X), np.int64)
        while at[0] < nodes:
            left = X[np.arange(len(X)), tree["fid"][at]] < tree["threshold"][at]
            at = 2 * at + 2 - left
        out.append(at - nodes)
    return np.array(out)


def tokens_of(arb, model, data, stride=None, n_rounds=-1, trees=None):
    trees = model.num_trees() if trees is None else trees
    stride = data.rows if stride is None else stride
    held = torch.full((trees, stride), -9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    leaves = model.leaf_tokens(data, held.data_ptr(), stride=stride, n_rounds=n_rounds)
    return held, leaves


@pytest.mark.parametrize("rows,features,rounds,depth,prebinned", [
    (1, 3, 2, 1, False), (63, 5, 3, 3, False), (3000, 9, 11, 6, False), (40_000, 30, 21, 5, False), (5000, 7, 5, 4, True),
    (900, 600, 3, 3, False)])
def test_leaf_tokens_are_the_walked_leaves(arb, rows, features, rounds, depth, prebinned):
    model, _, _, _, _ = make(arb, 0, rows=3000, features=features, rounds=rounds, depth=depth, prebinned=prebinned)
    rng = np.random.default_rng(rows)
    if prebinned:
        X = rng.integers(0, 64, size=(rows, features), dtype=np.uint8)
        data = arb.DMatrix(X, quantized=True)
    else:
        X = rng.normal(size=(rows, features)).astype(np.float32)
        X[rng.random(X.shape) < 0.1] = np.nan
        data = arb.DMatrix(X)
    want = walk(model, X.astype(np.float32)) + np.arange(rounds)[:, None] * 2 ** depth
    held, leaves = tokens_of(arb, model, data, stride=rows + 5)
    assert leaves == [rounds * 2 ** depth]
    assert np.array_equal(held[:, :rows].cpu().numpy(), want)
    assert (held[:, rows:] == -9).all()
    # the first two trees
    held, leaves = tokens_of(arb, model, data, n_rounds=2, trees=2)
    assert leaves == [2 * 2 ** depth] and np.array_equal(held.cpu().numpy(), want[:2])
    # what the booster answers is the lookup of its leaf weights
    held, leaves = tokens_of(arb, model, data)
    table = torch.tensor(np.concatenate([model.tree(t)["weights"] for t in range(rounds)])).cuda()
    out = torch.empty(rows, device="cuda")
    arb.embedding(out.data_ptr(), table.data_ptr(), held.data_ptr(), rows, leaves[0], 1, bag=rounds, token_stride=1, bag_stride=rows)
    magnitude = table.cpu().double()[held.cpu().long()].abs().sum(0).numpy() + 0.5
    off = np.abs(out.cpu().double().numpy() + 0.5 - model.predict(data).astype(np.float64))
    assert (off <= 2 * (rounds + 3) * U * magnitude).all()  # both are sums in float32


def test_leaf_tokens_of_several_classes_stand_by_class(arb):
    model, data, X, _, _ = make(arb, 4, classes=3, rounds=4)
    want = walk(model, X)
    order = [t for c in range(3) for t in range(c, 12, 3)]
    first = np.tile(np.arange(4) * 16, 3)[:, None]
    held, leaves = tokens_of(arb, model, data)
    assert leaves == [64, 64, 64]
    assert np.array_equal(held.cpu().numpy(), want[order] + first)
    # the model's sums are walked as before
    assert model.predict(data).shape == (3000, 3)


def test_leaf_tokens_of_a_streamed_matrix(arb):
    rng = np.random.default_rng(4)
    X = rng.integers(0, 64, size=(5000, 8), dtype=np.uint8)
    y = (X[:, 0].astype(np.float32) - 30) / 10
    config = {"objective": 0, "method": 1, "internals": {"hist_size": 64, "upload_features": False, "stream_block_rows": 1024},
              "tree": {"max_depth": 3, "eta": 0.3, "lambda": 1.0, "min_child_weight": 1.0}}
    data = arb.DMatrix(X, y=y, quantized=True)
    model = arb.train(config, data, 3)
    held, leaves = tokens_of(arb, model, data)
    assert np.array_equal(held.cpu().numpy(), walk(model, X.astype(np.float32)) + np.arange(3)[:, None] * 8)


def directions_64(objective, sums, init, y, labels):
    """Descent directions [classes][rows] in 64 bits."""
    if objective == 0:
        return y.astype(np.float64)[None] - (sums + init)
    if objective == 1:
        return y.astype(np.float64)[None] - 1 / (1 + np.exp(-(sums + init)))
    e = np.exp(sums - sums.max(0))
    p = e / e.sum(0)
    return (labels[None] == np.arange(len(sums))[:, None]) - p


@pytest.mark.parametrize("objective,classes", [(0, 1), (1, 1), (4, 3)])
def test_one_step_of_refinement(arb, objective, classes):
    model, data, X, y, labels = make(arb, objective, classes=classes, rounds=5)
    n, trees = len(X), model.num_trees()
    leaf = walk(model, X)
    before = [model.tree(t)["weights"].astype(np.float64) for t in range(trees)]
    sums, size = np.zeros((classes, n)), np.zeros((classes, n))
    for t in range(trees):
        sums[t % classes] += before[t][leaf[t]]
        size[t % classes] += np.abs(before[t][leaf[t]])
    d = directions_64(objective, sums, {0: 0.5, 1: 0.0, 4: 0.0}[objective], y, labels)
    # a direction is off by the lookup's sum, and by a few roundings of values around 1 (slopes of the links are at most 1)
    per = trees // classes
    dd = (per + 3) * U * size.sum(0) + 8 * U * (1 + np.abs(sums).max(0) + np.abs(d).max(0))
    lr, eps, decay = 0.01, 1e-3, 0.1
    plain = model.predict(data)
    model.refine_leaves(steps=1, lr=lr, eps=eps, weight_decay=decay)
    for t in range(trees):
        g = np.zeros(len(before[t]))
        np.add.at(g, leaf[t], -d[t % classes] / n)
        dg, count = np.zeros_like(g), np.bincount(leaf[t], minlength=len(g))
        np.add.at(dg, leaf[t], dd / n)
        mag = np.zeros_like(g)
        np.add.at(mag, leaf[t], np.abs(d[t % classes]) / n)
        dg += (count + 4) * U * mag
        want = before[t] * (1 - lr * decay) - lr * g / (np.abs(g) + eps)
        bound = lr * dg / eps + 16 * U * lr + 3 * U * np.abs(before[t])
        got = model.tree(t)["weights"].astype(np.float64)
        assert (np.abs(got - want) <= bound).all(), t
    assert not np.array_equal(plain, model.predict(data))


def test_many_steps_are_the_operators_one_after_the_other(arb):
    model, data, X, y, _ = make(arb, 0, rows=5000, rounds=9, depth=5)
    other = arb.load(model.dump())
    n, trees, steps, lr = len(X), 9, 12, 0.02
    held, (leaves,) = tokens_of(arb, model, data)
    weights = torch.tensor(np.concatenate([model.tree(t)["weights"] for t in range(trees)])).cuda()
    grad, m, v = torch.empty_like(weights), torch.zeros_like(weights), torch.zeros_like(weights)
    out, target = torch.empty(n, device="cuda"), torch.tensor(y).cuda()
    pairs = torch.empty(2, n * trees, dtype=torch.int32, device="cuda")
    size = max(arb.embedding_sort_bytes(n, leaves, bag=trees), arb.embedding_grad_bytes(n, 1, bag=trees))
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    arb.embedding_sort(pairs[0].data_ptr(), pairs[1].data_ptr(), held.data_ptr(), n, leaves, work.data_ptr(), size, bag=trees,
                       token_stride=1, bag_stride=n)
    for step in range(1, steps + 1):
        arb.embedding(out.data_ptr(), weights.data_ptr(), held.data_ptr(), n, leaves, 1, bag=trees, token_stride=1, bag_stride=n)
        d = target - (out + 0.5)
        arb.embedding_grad(grad.data_ptr(), d.data_ptr(), pairs[0].data_ptr(), pairs[1].data_ptr(), n, leaves, 1, work.data_ptr(),
                           size, bag=trees, scale=-1.0 / n)
        arb.adamw([weights.data_ptr()], [grad.data_ptr()], [m.data_ptr()], [v.data_ptr()], [leaves], step, lr, weight_decay=0.0)
    model.refine_leaves(steps=steps, lr=lr)
    assert np.array_equal(np.concatenate([model.tree(t)["weights"] for t in range(trees)]), weights.cpu().numpy())
    # predictions and the model's text are those of the new weights, on the device as on the host
    after = model.predict(data)
    model.predict_on_device(False)
    assert np.array_equal(after, model.predict(data))
    assert np.array_equal(arb.load(model.dump()).predict(data), after)
    # a loaded booster refines on a matrix of the caller's, to the same weights
    other.refine_leaves(data, steps=steps, lr=lr)
    assert np.array_equal(other.predict(data), after)


def test_no_steps_change_nothing(arb):
    model, data, _, _, _ = make(arb, 1)
    before = model.predict(data)
    model.refine_leaves(steps=0)
    assert np.array_equal(model.predict(data), before)


def test_refusals(arb):
    model, data, X, y, _ = make(arb, 0, rows=500, rounds=2)
    held = torch.empty(2, 500, dtype=torch.int32, device="cuda")
    with pytest.raises(arb.ArboretumError, match="stride"):
        model.leaf_tokens(data, held.data_ptr(), stride=499)
    with pytest.raises(arb.ArboretumError, match="token array"):
        model.leaf_tokens(data, None)
    with pytest.raises(arb.ArboretumError, match="no trees"):
        model.leaf_tokens(data, held.data_ptr(), n_rounds=0)
    with pytest.raises(arb.ArboretumError, match="no trees"):
        arb.Garden(model.config, data).refine_leaves()
    with pytest.raises(arb.ArboretumError, match="y is not set"):
        model.refine_leaves(arb.DMatrix(X))
    bad = y.copy()
    bad[3] = np.nan
    with pytest.raises(arb.ArboretumError, match="finite"):
        model.refine_leaves(arb.DMatrix(X, y=bad))
    with pytest.raises(arb.ArboretumError, match="steps"):
        model.refine_leaves(steps=-1)
    weights = model.tree(0)["weights"].copy()
    with pytest.raises(arb.ArboretumError, match="must not be negative"):
        model.refine_leaves(lr=-1.0)
    assert np.array_equal(model.tree(0)["weights"], weights)
    model.grow_tree()  # what was refused left the booster as it was
    model.refine_leaves(steps=1)
    with pytest.raises(arb.ArboretumError, match="refined"):
        model.grow_tree()
    assert model.num_trees() == 3
